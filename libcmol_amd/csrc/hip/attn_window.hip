// attn_window.hip — attention over a sliding window with sinks, one wave per
// (query head, item).
#include "attn_rows.h"

template <int DH, typename KT, bool SHARED>
__global__ __launch_bounds__(256) void k_rows_wave(RowsArgs a)
{
#pragma clang fp contract(off)
    constexpr int DL = RowState<DH>::DL;
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (long)a.n * a.n_heads) return;
    const int i = (int)(row / a.n_heads), h = (int)(row % a.n_heads), kvh = h / (a.n_heads / a.n_kv);
    const bool on = lane * DL < DH;
    RowState<DH> r;
    r.m = -INFINITY;
    r.l = 0.0f;
    const size_t at = (size_t)row * DH + (on ? lane * DL : 0);
#pragma unroll
    for (int d = 0; d < DL; d++) {
        r.q[d] = a.q[at + d];
        r.o[d] = 0.0f;
    }
    size_t base;
    const int L = rows_item(a, i, &base);
    base += (size_t)kvh * a.max_ctx * DH;
    const KT *k = (const KT *)a.k + base, *v = (const KT *)a.v + base;
    int seen = L;
    if constexpr (SHARED) {
        const size_t pb = (size_t)kvh * a.prefix_ctx * DH;
        row_walk<DH, KT>(r, (const KT *)a.pk + pb, (const KT *)a.pv + pb, 0, a.prefix);
        row_walk<DH, KT>(r, k, v, 0, L);
        seen += a.prefix;
    } else {
        const int s = min(a.sinks, L);
        row_walk<DH, KT>(r, k, v, 0, s);
        row_walk<DH, KT>(r, k, v, max(s, L - a.window), L);
    }
    if (!on) return;
#pragma unroll
    for (int d = 0; d < DL; d++) a.out[at + d] = seen > 0 ? r.o[d] / r.l : 0.0f;
}

template <bool SHARED>
static int launch_rows(const RowsArgs &a, hipStream_t s)
{
    const dim3 grid((unsigned)(((long)a.n * a.n_heads + 3) / 4)), block(256);
#define ROWS(DHV)                                                                                        \
    if (a.kv_f16) hipLaunchKernelGGL((k_rows_wave<DHV, _Float16, SHARED>), grid, block, 0, s, a);        \
    else hipLaunchKernelGGL((k_rows_wave<DHV, float, SHARED>), grid, block, 0, s, a);
    switch (a.d_head) {
    case 16: ROWS(16); break;
    case 32: ROWS(32); break;
    case 64: ROWS(64); break;
    case 128: ROWS(128); break;
    case 256: ROWS(256); break;
    default: return -4;
    }
#undef ROWS
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

int launch_attn_window(const RowsArgs &a, hipStream_t s) { return launch_rows<false>(a, s); }
int launch_attn_shared(const RowsArgs &a, hipStream_t s) { return launch_rows<true>(a, s); }
