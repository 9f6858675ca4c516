// logits.hip — penalties for repeated tokens, biases, grammar masks and the
// greedy choice on rows of logits.  Token v of a row with c occurrences in the
// row's history:
//   x1 = c times: x > 0 ? x / repeat : x * repeat      (repeat > 1)
//   x2 = x1 - (frequency c + presence)                  (c > 0)
//   x3 = x2 + bias
//   x4 = allowed ? x3 : -inf
// The repeat penalty is applied an occurrence at a time, each result rounded
// to fp32, as cmol_apply_repeat_penalty does.
//
// One work-group per (slab of SLAB tokens, row): the slab's occurrences are
// counted in LDS from the row's whole history (integer counts: the order of
// the atomics does not matter), and of a token's bias entries the last is kept
// (a maximum over their places).  The largest (value, lowest token) of a slab
// goes to `part`; k_logits_pick takes the row's.
#include "logits.h"

constexpr int SLAB = 2048;

int logits_slabs(int vocab) { return (vocab + SLAB - 1) / SLAB; }

__device__ inline unsigned long long key_max(unsigned long long k)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t hi = __shfl_xor((uint32_t)(k >> 32), o, 64), lo = __shfl_xor((uint32_t)k, o, 64);
        const unsigned long long x = ((unsigned long long)hi << 32) | lo;
        k = x > k ? x : k;
    }
    return k;
}

__global__ __launch_bounds__(256) void k_logits(LogitsArgs a)
{
#pragma clang fp contract(off)
    __shared__ int cnt[SLAB], last[SLAB];
    __shared__ unsigned long long best[4];
    const int row = blockIdx.y, v0 = blockIdx.x * SLAB, nv = min(SLAB, a.vocab - v0), tid = threadIdx.x;
    const int hl = a.history ? min(max(a.history_len[row], 0), a.history_cap) : 0;
    const int bl = a.bias_ids ? min(max(a.bias_len[row], 0), a.bias_cap) : 0;
    const int32_t *hist = a.history + (size_t)row * a.history_cap;
    const int32_t *bids = a.bias_ids + (size_t)row * a.bias_cap;
    const float *bias = a.bias + (size_t)row * a.bias_cap;
    for (int i = tid; i < SLAB; i += 256) cnt[i] = last[i] = 0;
    __syncthreads();
    for (int i = tid; i < hl; i += 256) {
        const unsigned u = (unsigned)(hist[i] - v0);
        if (hist[i] >= 0 && u < (unsigned)nv) atomicAdd(&cnt[u], 1);
    }
    for (int i = tid; i < bl; i += 256) {
        const unsigned u = (unsigned)(bids[i] - v0);
        if (bids[i] >= 0 && u < (unsigned)nv) atomicMax(&last[u], i + 1);
    }
    __syncthreads();
    const float rep = a.repeat ? a.repeat[row] : 1.0f;
    const float frq = a.frequency ? a.frequency[row] : 0.0f, prs = a.presence ? a.presence[row] : 0.0f;
    const int mr = !a.mask ? -1 : a.mask_row ? a.mask_row[row] : row;
    const bool masked = mr >= 0 && mr < a.mask_rows;
    const uint32_t *mask = a.mask + (masked ? (size_t)mr * ((a.vocab + 31) / 32) : 0);
    unsigned long long top = 0;
    for (int i = tid; i < nv; i += 256) {
        const int v = v0 + i;
        float x = a.x[row * a.stride + v];
        const int c = cnt[i];
        if (rep > 1.0f) {
            for (int j = 0; j < c; j++) {
                const float y = x > 0.0f ? x / rep : x * rep;
                if (y == x) break;   // 0 or an infinity: every further one leaves it
                x = y;
            }
        }
        if (c) x -= frq * (float)c + prs;
        if (last[i]) x += bias[last[i] - 1];
        if (masked && !((mask[v >> 5] >> (v & 31)) & 1)) x = -INFINITY;
        if (a.out) a.out[row * a.stride + v] = x;
        if (x > -INFINITY) top = max(top, argmax_key(x + 0.0f, (uint32_t)v));   // (never a NaN; -0 as 0)
    }
    if (!a.next) return;
    top = key_max(top);
    if ((tid & 63) == 0) best[tid >> 6] = top;
    __syncthreads();
    if (tid == 0) a.part[(size_t)row * gridDim.x + blockIdx.x] = max(max(best[0], best[1]), max(best[2], best[3]));
}

__global__ __launch_bounds__(64) void k_logits_pick(LogitsArgs a, int slabs)
{
    const int row = blockIdx.x;
    unsigned long long top = 0;
    for (int i = threadIdx.x; i < slabs; i += 64) top = max(top, a.part[(size_t)row * slabs + i]);
    top = key_max(top);
    if (threadIdx.x == 0) a.next[row] = top ? (int)argmax_index(top) : -1;
}

int launch_logits(const LogitsArgs &a, hipStream_t s)
{
    const int slabs = logits_slabs(a.vocab);
    hipLaunchKernelGGL(k_logits, dim3(slabs, a.n), dim3(256), 0, s, a);
    if (a.next) hipLaunchKernelGGL(k_logits_pick, dim3(a.n), dim3(64), 0, s, a, slabs);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
