// attn_window.hip — attention over a sliding window with sinks (attn_rows.h):
// single tokens of many sessions, and consecutive tokens of one.  Single tokens
// behind a short shared prefix (attn_shared.hip) are single tokens whose first
// run of positions is in another cache.
#include "attn_rows.h"

#include <cstdlib>

// ---- single tokens ---------------------------------------------------------------

// Work-group of NW waves (16 query heads of a kv head, slot): the piece of that
// slot, or item `slot` whole where there are no pieces.  Bound by the cache's bytes
// where there are enough (32 sessions of 16/4 heads of 128 over fp16, windows of
// 4096, 176 MB: 33.9 us, 5.2 TB/s), else by a launch and its dependent loads (one
// session, a window of 128: 5.1 us).
template <int DH, typename KT, int NW, bool FEW, bool NT>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(DH == 256 ? 1 : 2))) void k_window(RowsArgs a)
{
#pragma clang fp contract(off)
    constexpr int TP = FEW ? FEW_TP : rw_tp<KT>();
    __shared__ typename std::conditional<FEW, FewMeet<DH, NW>, RowsMeet<DH, NW>>::type meet;
    const int G = a.n_heads / a.n_kv, blocks = (G + 15) / 16;
    const int kvh = blockIdx.x / blocks, r0 = (blockIdx.x % blocks) * 16, slot = blockIdx.y;
    const int tid = threadIdx.x, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const RowsPiece p = rows_piece<TP>(a, slot);
    if (p.item < 0) return;
    RowsLine<TP> line = rows_line<TP>(p.L - 1, p.L - 1, a.window, a.sinks);
    int u1 = p.u1;
    if (a.prefix) {
        line.s = a.prefix;
        line.ns = (a.prefix + TP - 1) / TP;
        u1 = line.tiles();
    }
    const bool none = u1 == 0;   // (a whole item's)
    const size_t row0 = (size_t)p.item * a.n_heads + (size_t)kvh * G;
    typename std::conditional<FEW, RowsFew<DH>, RowsWave<DH, KT, 1>>::type w;
    w.load([&](int r) { return a.q + (row0 + min(r0 + r, G - 1)) * DH; });
    const size_t base = (p.L > 0 ? (size_t)p.slot * a.slot_stride : 0) + (size_t)kvh * a.max_ctx * DH;
    RowsFrom<KT> from((const KT *)a.k + base, (const KT *)a.v + base);
    if (a.prefix) {
        from.k1 = (const KT *)a.pk + (size_t)kvh * a.prefix_ctx * DH;
        from.v1 = (const KT *)a.pv + (size_t)kvh * a.prefix_ctx * DH;
    }
    if constexpr (FEW) few_walk<DH, NT>(w, from, line, p.u0 + wid, u1, NW);
    else rows_walk<DH, KT, 1, false, NT>(w, from, line, p.u0 + wid, u1, NW, nullptr);
    const size_t part = ((size_t)kvh * rows_slots(a) + slot) * G;
    auto put = [&](int r, float m, float l, int d, auto &x) {
        r += r0;
        if (r >= G) return;
        if (p.whole) {
            const float f = none ? 0.0f : 1.0f / l;
            for (auto &y : x) y = none ? 0.0f : y * f;
            rows_store(a.out + (row0 + r) * DH + d, x);
        } else {
            rows_store(a.po + (part + r) * DH + d, x);
            if (d == 0) {
                a.pm[part + r] = m;
                a.pl[part + r] = l;
            }
        }
    };
    if constexpr (FEW) few_finish(w, meet, put);
    else rows_finish(w, meet, put);
}

// One work-group per (query head, item): the item's pieces.  A launch and two
// dependent loads: 4.7 us for 32 items of 16 heads.
template <int DH, int TP>
__global__ __launch_bounds__(256) void k_window_merge(RowsArgs a)
{
    constexpr int LPR = DH / 4;
    const int G = a.n_heads / a.n_kv, h = blockIdx.x, kvh = h / G, i = blockIdx.y, tid = threadIdx.x;
    int first;
    const int np = rows_pieces<TP>(a, i, &first);
    if (np == 1) return;   // finished by its only piece
    const size_t p0 = ((size_t)kvh * rows_slots(a) + first) * G + h % G;
    const f32x4 o = rows_sum<DH, 256 / LPR, 4>(np, tid % LPR, tid / LPR, [&](int j, const float **m, const float **l, const float **x) {
        const size_t at = p0 + (size_t)j * G;
        *m = a.pm + at;
        *l = a.pl + at;
        *x = a.po + at * DH;
    });
    if (tid < LPR) *(f32x4 *)(a.out + ((size_t)i * a.n_heads + h) * DH + 4 * tid) = o;
}

// ---- prompts ---------------------------------------------------------------------

// Rows of a kv head are (token, head of the group), token-major, in blocks of
// 16; work-group (block and kv head, part) walks its part of the tiles that the
// block's tokens see between them.  For prompts of few rows: 45 tokens of 9/3 heads
// of 64 over fp32, window 256, 7.9 us, of which a launch is about half.
template <int DH, typename KT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DH == 256 ? 1 : 2))) void k_window_prompt(RowsArgs a)
{
#pragma clang fp contract(off)
    constexpr int TP = rw_tp<KT>(), NW = 4;
    __shared__ RowsMeet<DH, NW> meet;
    __shared__ int odd, odd_row[16];
    const int G = a.n_heads / a.n_kv, rows = a.n * G, blocks = gridDim.x / a.n_kv;
    // the blocks of the longest lines first
    const int kvh = blockIdx.x % a.n_kv, r0 = (blocks - 1 - (int)(blockIdx.x / a.n_kv)) * 16, part = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nr = min(16, rows - r0);
    RowsSeen seen;
    seen.first = a.pos0 + r0 / G;
    seen.last = a.pos0 + (r0 + nr - 1) / G;
    seen.window = a.window;
    seen.sinks = a.sinks;
    const RowsLine<TP> line = rows_line<TP>(seen.first, seen.last, a.window, a.sinks);
    const int T = line.tiles(), R = (T + a.parts - 1) / a.parts;
    const int u0 = min(part * R, T), u1 = min(u0 + R, T);
    const int pos = a.pos0 + min(r0 + (lane & 15), rows - 1) / G;
    seen.pos = &pos;
    auto row_at = [&](int r) {   // of q and out
        r = min(r0 + r, rows - 1);
        return (size_t)(r / G) * a.n_heads + (size_t)kvh * G + r % G;
    };
    const size_t base = (size_t)kvh * a.max_ctx * DH;
    const KT *k = (const KT *)a.k + base, *v = (const KT *)a.v + base;
    RowsWave<DH, KT, 1> w;
    w.load([&](int r) { return a.q + row_at(r) * DH; });
    if (tid == 0) odd = 0;
    if (tid < 16) odd_row[tid] = 0;
    __syncthreads();
    rows_walk<DH, KT, 1, true, false>(w, RowsFrom<KT>(k, v), line, u0 + wid, u1, NW, &seen);
    const size_t x0 = ((size_t)kvh * rows + r0) * a.parts + part;   // + r * parts
    rows_finish(w, meet, [&](int r, float m, float l, int d, auto &x) {
        if (r >= nr) return;
        float z = l * 0.0f;
        for (auto &y : x) z += y * 0.0f;
        if (!(z == 0.0f)) odd = odd_row[r] = 1;
        if (a.parts == 1) {
            const float f = 1.0f / l;
            for (auto &y : x) y *= f;
            rows_store(a.out + row_at(r) * DH + d, x);
        } else {
            const size_t at = x0 + (size_t)r * a.parts;
            rows_store(a.xo + at * DH + d, x);
            if (d == 0) {
                a.xm[at] = m;
                a.xl[at] = l;
            }
        }
    });
    // A masked position is in its tile's products with weight 0, which a V row
    // that is not finite turns into NaN for the rows that do not see it: rows
    // whose outputs are not finite are walked again one by one.
    __syncthreads();
    if (!odd) return;
    constexpr int DL = RowState<DH>::DL;
    const bool on = lane * DL < DH;
    for (int r = wid; r < nr; r += NW) {
        if (!odd_row[r]) continue;
        const size_t qa = row_at(r) * DH + (on ? lane * DL : 0);
        const int p = a.pos0 + (r0 + r) / G;
        RowState<DH> t;
        t.m = -INFINITY;
        t.l = 0.0f;
#pragma unroll
        for (int d = 0; d < DL; d++) {
            t.q[d] = a.q[qa + d];
            t.o[d] = 0.0f;
        }
        for (int u = u0; u < u1; u++) {
            int p0, cnt;
            line.tile(u, &p0, &cnt);
            const int end = min(p0 + cnt, p + 1), lo = p + 1 - a.window;
            row_walk<DH, KT>(t, k, v, p0, min(end, a.sinks));
            row_walk<DH, KT>(t, k, v, max(max(p0, lo), min(a.sinks, end)), end);
        }
        if (!on) continue;
        const size_t at = x0 + (size_t)r * a.parts;
#pragma unroll
        for (int d = 0; d < DL; d++) {
            if (a.parts == 1) a.out[qa + d] = t.o[d] / t.l;
            else a.xo[at * DH + lane * DL + d] = t.o[d];
        }
        if (a.parts > 1 && lane == 0) {
            a.xm[at] = t.m;
            a.xl[at] = t.l;
        }
    }
}

// The parts of (query head, token) rows, a lane per four dimensions.  Bound by the
// partial results: five parts of 700 tokens of 16 heads of 128, 29 MB, in 7.0 us.
template <int DH>
__global__ __launch_bounds__(256) void k_prompt_parts(RowsArgs a)
{
    constexpr int LPR = DH / 4;
    const size_t row = (size_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;   // of out
    if (row >= (size_t)a.n * a.n_heads) return;
    const int G = a.n_heads / a.n_kv, t = (int)(row / a.n_heads), h = (int)(row % a.n_heads), d4 = threadIdx.x % LPR;
    const size_t x0 = ((size_t)(h / G) * a.n * G + (size_t)t * G + h % G) * a.parts;
    const f32x4 o = rows_sum<DH, 1, 8>(a.parts, d4, 0, [&](int j, const float **m, const float **l, const float **x) {
        *m = a.xm + x0 + j;
        *l = a.xl + x0 + j;
        *x = a.xo + (x0 + j) * DH;
    });
    *(f32x4 *)(a.out + row * DH + 4 * d4) = o;
}

// ---- plans and launches ------------------------------------------------------------

// Most tiles of a token's line.
static long span_tiles(int max_ctx, int window, int sinks)
{
    const long w = std::min(window, max_ctx), s = std::min(sinks, max_ctx);
    return std::min((long)ceil_div(w, RW_PLAN_TP) + ceil_div(s, RW_PLAN_TP), (long)ceil_div(max_ctx, RW_PLAN_TP) + 2);
}

int rows_whole_env()
{
    const char *e = getenv("CMOL_SESSION_WHOLE");
    return e && (e[0] == '0' || e[0] == '1') ? e[0] - '0' : -1;
}

int rows_plan_bal(int n, long heads, long span, long wgs)
{
    if (n * heads >= RW_WGS || n * span > INT32_MAX / 4) return 0;
    return (int)std::max(std::min(wgs / heads, n * (long)ceil_div(span, RW_RMIN)), 2L * n);
}

// Whether every item is one work-group's: no merge launch and no search, but the
// longest item is the call's time.  By what both are estimated to cost at most,
// the pieces' bytes at six tenths of what they may be, and up to WIN_RISK
// microseconds (a batch whose sessions are short but for one costs as much, where
// pieces would take 9).  Fitted to 1 .. 64 sessions of 16/4 heads of 128 and 9/3 of
// 64, windows of 300 .. 4000; both sides measured, in pieces and whole: one session
// of 16/4, fp32, window 900: 8.8 and 15.6 us, of 9/3, fp16: 8.5 and 8.0; 16 of 9/3, fp32,
// 1400: 13.6 and 12.9; 64 of 9/3, fp16, 2000: 24.2 and 18.0.
constexpr double WIN_RISK = 16;
static bool window_whole(int n, int n_heads, int n_kv, int d_head, int max_ctx, int window, int sinks, int kv_f16)
{
    const int e = rows_whole_env();
    if (e >= 0) return e;
    const double heads = (double)n_kv * ceil_div(n_heads / n_kv, 16), row = d_head * (kv_f16 ? 4 : 8);
    const double seen = std::min((double)max_ctx, (double)std::min(window, max_ctx) + std::min(sinks, max_ctx));
    const double together = rows_together(n * heads, seen, d_head, kv_f16);
    return together < WIN_RISK && together < 8 + 0.008 * n * n_kv + 0.6 * n * heads * seen * row / 5.6e6;
}

RowsPlan rows_plan_window(int n, int n_heads, int n_kv, int d_head, int max_ctx, int window, int sinks)
{
    RowsPlan p;
    const int G = n_heads / n_kv;
    if (!window_whole(n, n_heads, n_kv, d_head, max_ctx, window, sinks, 0) ||
        !window_whole(n, n_heads, n_kv, d_head, max_ctx, window, sinks, 1))
        p.bal = rows_plan_bal(n, (long)n_kv * ceil_div(G, 16), span_tiles(max_ctx, window, sinks), RW_WGS);
    if (p.bal) p.pieces = (size_t)n_kv * p.bal * G;
    return p;
}

// A prompt's form and the parts of its positions by what they are estimated to
// cost, in microseconds: work-groups of 16 rows that read the cache themselves
// (k_window_prompt), or of 128 that share it through LDS (attn_wprompt.hip).
// Fitted to prompts of 16 .. 4096 tokens of 16/4 heads of 128 and 15/5 of 64
// behind 5000 positions, windows of 128 .. 2048: the start and end of a
// work-group, a tile's step (the matrix and vector instructions of the
// work-groups that share a CU add up), the merge's launch and traffic.  Both
// sides measured: 256 tokens, window 2048, fp16: 30 us by itself, 36 shared; 700:
// 63, 46; 64 tokens, fp32: 24, 36; 500: 84, 51.
struct PromptForm {
    bool lds = false;
    int parts = 1;
    double us = 0;
};
static PromptForm prompt_form(bool lds, int n, int n_heads, int n_kv, int d_head, long ctx, int window, int sinks, int kv_f16)
{
    const int G = n_heads / n_kv, rows = lds ? WP_ROWS : 16, tp = lds || kv_f16 ? 32 : 16;
    const long blocks = (long)n_kv * ceil_div((long)n * G, rows);
    const long seen = std::min(ctx, std::min((long)window, ctx) + std::min((long)sinks, ctx) + std::min(n, rows / G + 1));
    const long tiles = ceil_div(seen, tp) + 1;
    const double dh = std::max(d_head, 32) / 128.0, traffic = (double)n * n_heads * d_head * 8 / 5e6;
    double fixed = 0;
    if (lds && !kv_f16) fixed = 4 + (double)std::min(ctx, (long)window + sinks + n) * n_kv * d_head * 16 / 4e6;   // the split copy
    PromptForm best;
    for (int p = 1; p <= 16 && p <= tiles; p++) {
        const double wgs = (double)blocks * p, deep = ceil_div(blocks * p, 256);   // (of the fullest CU)
        double us = fixed + (p > 1 ? 4.0 + p * traffic : 0.0);
        if (lds) us += 8.0 * std::max(1.0, wgs / 512) + ceil_div(tiles, p) * (kv_f16 ? 1.0 : 1.55) * std::max(0.5 + 0.6 * dh, (0.16 + 0.64 * dh) * deep);
        else us += 6.0 * std::max(1.0, wgs / 1024) + ceil_div(ceil_div(tiles, p), 4) * (kv_f16 ? 0.15 + 0.95 * dh : 0.25 + dh) * deep;
        if (p == 1 || us < best.us) {
            best.parts = p;
            best.us = us;
        }
    }
    best.lds = lds;
    return best;
}
// (CMOL_WINDOW_PROMPT=0 / 1: the first form / the second wherever it runs)
static PromptForm prompt_best(int n, int n_heads, int n_kv, int d_head, long ctx, int window, int sinks, int kv_f16)
{
    const PromptForm a = prompt_form(false, n, n_heads, n_kv, d_head, ctx, window, sinks, kv_f16);
    const char *e = getenv("CMOL_WINDOW_PROMPT");
    if (!wprompt_takes(d_head) || (e && e[0] == '0')) return a;
    const PromptForm b = prompt_form(true, n, n_heads, n_kv, d_head, ctx, window, sinks, kv_f16);
    return b.us < a.us || (e && e[0] == '1') ? b : a;
}

RowsPlan rows_plan_prompt(int n, int n_heads, int n_kv, int d_head, int max_ctx, int window, int sinks)
{
    RowsPlan p;
    for (int f16 = 0; f16 < 2; f16++) {
        const PromptForm f = prompt_best(n, n_heads, n_kv, d_head, max_ctx, window, sinks, f16);
        p.parts = std::max(p.parts, f.parts);
        if (f.lds && !f16) p.split = wprompt_split_bytes(n, n_kv, d_head, max_ctx, window, sinks);
    }
    if (p.parts > 1) p.cross = (size_t)n * n_heads * p.parts;
    return p;
}

// Whether the caches are streamed past the L2s: where a call may read so much that
// nothing of a cache is there again when the next call comes.  Three sets of caches
// in turn, plain and streamed: 32 sessions of 16/4 heads of 128, windows of 4096 (268
// MB at most) fp32 68.7 and 60.6 us, fp16 40.0 and 39.0; windows of 2000 over fp16
// (131 MB) 29.1 and 27.8; 1400 (92 MB) 21.5 and 26.5.
static bool window_stream(const RowsArgs &a)
{
    const double seen = std::min((double)a.max_ctx, (double)a.window + a.sinks);
    return !a.prefix && seen * a.n * a.n_kv * a.d_head * (a.kv_f16 ? 4 : 8) > 110e6;
}

int launch_attn_window(const RowsArgs &a0, hipStream_t s)
{
    RowsArgs a = a0;
    if (a.prefix || window_whole(a.n, a.n_heads, a.n_kv, a.d_head, a.max_ctx, a.window, a.sinks, a.kv_f16)) a.bal = 0;
    const dim3 grid(a.n_kv * ceil_div(a.n_heads / a.n_kv, 16), rows_slots(a));
    // eight waves for items that have more than one round of tiles for four
    // (d_head 256: four, for their registers)
    const bool wide =
        !a.bal && a.d_head < 256 && span_tiles(a.max_ctx, a.window, a.sinks) + ceil_div(a.prefix, RW_PLAN_TP) > 4;
    const bool few = few_takes(a.d_head, a.n_heads / a.n_kv, a.kv_f16);
    const bool nt = window_stream(a);
#define LAUNCH(DH, KT, NW, FEW)                                                                      \
    {                                                                                                \
        if (DH >= 64 && nt) hipLaunchKernelGGL((k_window<DH, KT, NW, FEW, DH >= 64>), grid, dim3(NW * 64), 0, s, a); \
        else hipLaunchKernelGGL((k_window<DH, KT, NW, FEW, false>), grid, dim3(NW * 64), 0, s, a);   \
    }
#define WIN_NW(DH, NW)                                        \
    if constexpr (few_takes(DH, 1, 0))                        \
        if (few) LAUNCH(DH, float, NW, true)                  \
    if (a.kv_f16) LAUNCH(DH, _Float16, NW, false)             \
    else if (!few) LAUNCH(DH, float, NW, false)
#define WIN(DH)                                               \
    if constexpr (DH < 256)                                   \
        if (wide) { WIN_NW(DH, 8) }                           \
    if (!wide) { WIN_NW(DH, 4) }
    RW_BY_D_HEAD(a.d_head, WIN)
#undef WIN
#undef WIN_NW
#undef LAUNCH
    if (a.bal) {
#define MERGE(DH)                                                                                              \
    if (a.kv_f16 || few) hipLaunchKernelGGL((k_window_merge<DH, 32>), dim3(a.n_heads, a.n), dim3(256), 0, s, a);      \
    else hipLaunchKernelGGL((k_window_merge<DH, 16>), dim3(a.n_heads, a.n), dim3(256), 0, s, a);
        RW_BY_D_HEAD(a.d_head, MERGE)
#undef MERGE
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

int launch_attn_window_prompt(const RowsArgs &a0, hipStream_t s)
{
    RowsArgs a = a0;
    const int room = a.parts, seen = a.pos0 + a.n;
    // (what this position's tokens see may be less than the plan's most: within its room)
    PromptForm f = prompt_best(a.n, a.n_heads, a.n_kv, a.d_head, seen, a.window, a.sinks, a.kv_f16);
    if (f.lds) {
        a.parts = std::min(room, f.parts);
        // no room for the f16 pairs, or a refused LDS limit: the other form
        if ((!a.kv_f16 && !a.split) || launch_wprompt(a, s))
            f = prompt_form(false, a.n, a.n_heads, a.n_kv, a.d_head, seen, a.window, a.sinks, a.kv_f16);
    }
    if (!f.lds) {
        a.parts = std::min(room, f.parts);
        const dim3 grid(a.n_kv * ceil_div((long)a.n * (a.n_heads / a.n_kv), 16), a.parts), block(256);
#define PRO(DH)                                                                                  \
    if (a.kv_f16) hipLaunchKernelGGL((k_window_prompt<DH, _Float16>), grid, block, 0, s, a);     \
    else hipLaunchKernelGGL((k_window_prompt<DH, float>), grid, block, 0, s, a);
        RW_BY_D_HEAD(a.d_head, PRO)
#undef PRO
    }
    if (a.parts > 1) {
        const dim3 grid((unsigned)(((size_t)a.n * a.n_heads * a.d_head + 1023) / 1024)), block(256);
#define MERGE(DH) hipLaunchKernelGGL(k_prompt_parts<DH>, grid, block, 0, s, a);
        RW_BY_D_HEAD(a.d_head, MERGE)
#undef MERGE
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
