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
// One work-group per (slab of the vocabulary, row).  The slab's logits and mask
// words are requested first; meanwhile its occurrences are counted in LDS from
// the row's whole history (integer counts: the order of the atomics does not
// matter), and of a token's bias entries the last is kept (a maximum over their
// places).  The largest (value, lowest token) of a slab goes to `part` and
// k_logits_pick takes the row's.
//
// Bound: the logits read and written once, above the launches' few microseconds;
// every work-group reads the row's history, so where the rows alone give each CU
// one slabs are large (SLAB 8192 on 1024 threads), else small (2048 on 256).  One
// row of 49152: 4.6 us and 1.5 for the pick; 32 of 128256 with every part, 33 MB:
// 14.3 and 3.9, of which the divisions of the word repeated most are 2.8.
#include "logits.h"
#include "lanes.h"

// The largest key of a wave: the largest upper half, then the largest lower one
// among the lanes that have it.
__device__ inline unsigned long long key_max(unsigned long long k)
{
    auto most = [](uint32_t x) {
        auto f = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
        return lanes_pair<32>(
            lanes_pair<16>(lanes_pair<8>(lanes_pair<4>(lanes_pair<2>(lanes_pair<1>(x, f), f), f), f), f), f);
    };
    const uint32_t hi = most((uint32_t)(k >> 32)), lo = most((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0);
    return ((unsigned long long)hi << 32) | lo;
}

// 1 / rep in two parts, the first of them rounded.
struct Reciprocal {
    float hi, lo;
    __device__ explicit Reciprocal(float rep) : hi(1.0f / rep), lo(fmaf(-rep, hi, 1.0f) * hi) {}
};
// x / rep rounded, for 2^-60 <= x <= 2^100 and rep <= 2^30 (every step stays among
// the normal numbers): the product with both parts is off by its last rounding
// and 2^-23 ulp, so within one ulp, and then the remainder is exact and one
// correction by the rounded reciprocal rounds it as the division does (Markstein).
__device__ inline float divide_step(float x, float rep, Reciprocal y)
{
    const float q = fmaf(x, y.hi, x * y.lo);
    return fmaf(fmaf(-rep, q, x), y.hi, q);
}

// The repeat penalty of c occurrences.  Eight steps at a time where there are
// as many: a word that fills its history is a chain of hundreds of dependent
// steps on one lane (32 rows, 211 occurrences at most: 11 us with a check a step).
__device__ inline float repeat_penalty(float x, int c, float rep, Reciprocal y)
{
#pragma clang fp contract(off)
    if (x > 0.0f) {
        for (; c >= 8 && x >= 0x1p-28f && x <= 0x1p+100f && rep <= 16.0f; c -= 8)
#pragma unroll
            for (int i = 0; i < 8; i++) x = divide_step(x, rep, y);
        for (; c > 0 && x >= 0x1p-60f && x <= 0x1p+100f && rep <= 0x1p+30f; c--) x = divide_step(x, rep, y);
        for (; c > 0; c--) {
            const float q = x / rep;
            if (q == x) break;   // every further one leaves it
            x = q;
        }
        return x;
    }
    for (; c >= 8; c -= 8) {
        const float was = x;
#pragma unroll
        for (int i = 0; i < 8; i++) x *= rep;
        if (x == was) return x;
    }
    for (; c > 0; c--) x *= rep;
    return x;
}

template <int SLAB, int NT>
__global__ __launch_bounds__(NT) void k_logits(LogitsArgs a)
{
#pragma clang fp contract(off)
    constexpr int Q = SLAB / NT / 4;   // fours of tokens per thread
    __shared__ __attribute__((aligned(16))) int cnt[SLAB], last[SLAB];
    __shared__ unsigned long long best[NT / 64];
    const int row = blockIdx.y, v0 = blockIdx.x * SLAB, nv = min(SLAB, a.vocab - v0), tid = threadIdx.x;
    const int hl = a.history ? min(max(a.history_len[row], 0), a.history_cap) : 0;
    const int bl = a.bias_ids ? min(max(a.bias_len[row], 0), a.bias_cap) : 0;
    const int mr = !a.mask ? -1 : a.mask_row ? a.mask_row[row] : row;
    const bool masked = mr >= 0 && mr < a.mask_rows;
    const float rep = a.repeat ? a.repeat[row] : 1.0f;
    const float frq = a.frequency ? a.frequency[row] : 0.0f, prs = a.presence ? a.presence[row] : 0.0f;
    const float *px = a.x + row * a.stride + v0;
    float *po = a.out ? a.out + row * a.stride + v0 : nullptr;
    const bool wide = (((uintptr_t)px | (uintptr_t)po) & 15) == 0;   // (uniform; v0 is a multiple of four)
    const uint32_t *mask = a.mask + (masked ? (size_t)mr * ((a.vocab + 31) / 32) : 0) + v0 / 32;

    // this thread's tokens 4 (tid + NT q) .. +3 of the slab (past nv: not used)
    f32x4 x[Q];
    uint32_t mw[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) {
        const int i = 4 * (tid + NT * q);
        mw[q] = masked && i < nv ? mask[i >> 5] >> (i & 31) : ~0u;
        if (wide && i + 4 <= nv) x[q] = *(const f32x4 *)(px + i);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) x[q][e] = i + e < nv ? px[i + e] : 0.0f;
    }
    if (hl | bl) {   // (uniform)
        const u32x4 z = {};
#pragma unroll
        for (int q = 0; q < Q; q++) {
            *(u32x4 *)&cnt[4 * (tid + NT * q)] = z;
            if (bl) *(u32x4 *)&last[4 * (tid + NT * q)] = z;
        }
        __syncthreads();
        const int32_t *hist = a.history + (size_t)row * a.history_cap;
        auto count = [&](int id) {
            const unsigned u = (unsigned)(id - v0);
            if (id >= 0 && u < (unsigned)nv) atomicAdd(&cnt[u], 1);
        };
        int i = tid;
        for (; i + 3 * NT < hl; i += 4 * NT) {   // four loads in one round trip
            const int t0 = hist[i], t1 = hist[i + NT], t2 = hist[i + 2 * NT], t3 = hist[i + 3 * NT];
            count(t0);
            count(t1);
            count(t2);
            count(t3);
        }
        for (; i < hl; i += NT) count(hist[i]);
        const int32_t *ids = a.bias_ids + (size_t)row * a.bias_cap;
        for (int j = tid; j < bl; j += NT) {
            const int id = ids[j];
            const unsigned u = (unsigned)(id - v0);
            if (id >= 0 && u < (unsigned)nv) atomicMax(&last[u], j + 1);
        }
        __syncthreads();
    }
    const Reciprocal y(rep);
    const float *bias = a.bias + (size_t)row * a.bias_cap;
    unsigned long long top = 0;
#pragma unroll
    for (int q = 0; q < Q; q++) {
        const int i = 4 * (tid + NT * q);
        if (hl) {
            const u32x4 c4 = *(const u32x4 *)&cnt[i];
            if (c4[0] | c4[1] | c4[2] | c4[3]) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int c = (int)c4[e];
                    if (c && rep > 1.0f) x[q][e] = repeat_penalty(x[q][e], c, rep, y);
                    if (c) x[q][e] -= frq * (float)c + prs;
                }
            }
        }
        if (bl) {
            const u32x4 l4 = *(const u32x4 *)&last[i];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (l4[e]) x[q][e] += bias[l4[e] - 1];
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (!((mw[q] >> e) & 1)) x[q][e] = -INFINITY;
        if (po) {
            // (a large output does not stay in the L2s, whose write-back the next kernel
            // would wait for: 32 rows of 128256 16.3 us, 15.0 streamed)
            if (wide && i + 4 <= nv && SLAB > 2048) __builtin_nontemporal_store(x[q], (f32x4 *)(po + i));
            else if (wide && i + 4 <= nv) *(f32x4 *)(po + i) = x[q];
            else
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e < nv) po[i + e] = x[q][e];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {   // (never a NaN; -0 as 0)
            const unsigned long long k = argmax_key(x[q][e] + 0.0f, (uint32_t)(v0 + i + e));
            if (i + e < nv && x[q][e] > -INFINITY && k > top) top = k;
        }
    }
    if (!a.next) return;
    top = key_max(top);
    if ((tid & 63) == 0) best[tid >> 6] = top;
    __syncthreads();
    if (tid >= 64) return;
    top = key_max(tid < NT / 64 ? best[tid] : 0);
    if (tid == 0) a.part[(size_t)row * gridDim.x + blockIdx.x] = top;
}

__global__ __launch_bounds__(64) void k_logits_pick(LogitsArgs a, int slabs)
{
    const int row = blockIdx.x;
    unsigned long long top = 0;
    for (int i = threadIdx.x; i < slabs; i += 64) {
        const unsigned long long k = a.part[(size_t)row * slabs + i];
        top = k > top ? k : top;
    }
    top = key_max(top);
    if (threadIdx.x == 0) a.next[row] = top ? (int)argmax_index(top) : -1;
}

constexpr int SLAB_MIN = 2048, SLAB_MAX = 8192;

int logits_slabs(int vocab) { return (vocab - 1) / SLAB_MIN + 1; }

int launch_logits(const LogitsArgs &a, hipStream_t s)
{
    const int big = (a.vocab - 1) / SLAB_MAX + 1;
    const bool large = (long)big * a.n >= 256;
    const int slabs = large ? big : logits_slabs(a.vocab);
    if (large) hipLaunchKernelGGL((k_logits<SLAB_MAX, 1024>), dim3(slabs, a.n), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((k_logits<SLAB_MIN, 256>), dim3(slabs, a.n), dim3(256), 0, s, a);
    if (a.next) hipLaunchKernelGGL(k_logits_pick, dim3(a.n), dim3(64), 0, s, a, slabs);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
