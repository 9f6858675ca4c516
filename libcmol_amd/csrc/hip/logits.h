// logits.h — launcher of the logits stage (logits.hip).
#pragma once
#include "common.h"

struct LogitsArgs {
    int n, vocab;
    long stride;                    // elements from one row to the next
    const float *x;
    float *out;                     // or null
    int32_t *next;                  // or null
    const int32_t *history, *history_len;   // [n][history_cap], [n], or null
    int history_cap;
    const float *repeat, *frequency, *presence;   // [n] each, or null
    const int32_t *bias_ids, *bias_len;     // [n][bias_cap], [n], or null
    const float *bias;
    int bias_cap;
    const uint32_t *mask;           // [mask_rows][(vocab + 31) / 32], or null
    const int32_t *mask_row;        // [n], or null: row i has mask row i
    int mask_rows;
    unsigned long long *part;       // [n][slabs] argmax keys (next wanted)
};

// Most vocabulary slabs of a row.
int logits_slabs(int vocab);
int launch_logits(const LogitsArgs &a, hipStream_t s);
