// attn_rows.h — attention of query rows whose visible positions are not simply
// the first seqlen of their own cache: a sliding window with sinks
// (attn_window.hip) and a prefix shared by the sessions (attn_shared.hip).
// An item is a session's token or a prompt token; query row (item, h) of kv
// head h / G sees
//   window   t <= p and (t < sinks or t > p - window), p = its position
//   shared   the prefix's positions, then its own t < seqlen
// and out = sum_t softmax_t(q . k_t / sqrt(d_head)) v_t over them, 0 where
// there are none.  Every sum and softmax statistic is fp32.
#pragma once
#include "common.h"

struct RowsArgs {
    const float *q;            // [n][n_heads*d_head]
    float *out;                // [n][n_heads*d_head]
    const void *k, *v;         // caches [slot][n_kv][max_ctx][d_head]
    size_t slot_stride;        // elements from one cache to the next
    const int32_t *slots;      // cache of each item (below 0: none), or null: item i has cache i
    const int32_t *seqlen;     // positions of each item's cache up to its own; null: pos0 + item + 1
    int n, n_heads, n_kv, d_head, max_ctx, kv_f16;
    int window, sinks;         // at most max_ctx each
    int pos0;                  // prompt: position of item 0 (seqlen null)
    const void *pk, *pv;       // shared prefix [n_kv][prefix_ctx][d_head]
    int prefix, prefix_ctx;
};

// Positions of item i's cache up to its own (0: it sees nothing there), and
// that cache.
__device__ __forceinline__ int rows_item(const RowsArgs &a, int i, size_t *base)
{
    if (!a.seqlen) {
        *base = 0;
        return a.pos0 + i + 1;
    }
    const int slot = a.slots ? a.slots[i] : i;
    *base = slot < 0 ? 0 : (size_t)slot * a.slot_stride;
    return slot < 0 ? 0 : max(min(a.seqlen[i], a.max_ctx), 0);
}

// One query row on one wave: lane l holds dimensions DL l .. +DL-1 (the first
// d_head lanes below 64).
template <int DH>
struct RowState {
    static constexpr int DL = DH < 64 ? 1 : DH / 64;
    float q[DL], o[DL], m, l;
};

// Positions t0 .. t1-1 of the cache rows at k and v into a row's online
// softmax, one position at a time.
template <int DH, typename KT>
__device__ void row_walk(RowState<DH> &r, const KT *k, const KT *v, int t0, int t1)
{
#pragma clang fp contract(off)
    constexpr int DL = RowState<DH>::DL;
    const int lane = threadIdx.x & 63;
    const bool on = lane * DL < DH;
    for (int t = t0; t < t1; t++) {
        const size_t at = (size_t)t * DH + (on ? lane * DL : 0);
        float s = 0.0f;
#pragma unroll
        for (int d = 0; d < DL; d++) s = fmaf(r.q[d], (float)k[at + d], s);
        s = wave_sum(on ? s : 0.0f) * (1.0f / sqrtf((float)DH));
        const float mn = fmaxf(r.m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float al = expf(r.m - ref), e = expf(s - ref);
        r.m = s != s ? s : mn;   // (fmaxf drops a NaN)
        r.l = r.l * al + e;
#pragma unroll
        for (int d = 0; d < DL; d++) r.o[d] = r.o[d] * al + e * (float)v[at + d];
    }
}

int launch_attn_window(const RowsArgs &a, hipStream_t s);
int launch_attn_shared(const RowsArgs &a, hipStream_t s);
