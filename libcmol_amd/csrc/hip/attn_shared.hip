// attn_shared.hip — decode attention of sessions that share a prefix
// (attn_rows.h).  The prefix is read once for all of them: per kv head the
// sessions' query rows (n G of them, session-major) form tiles of 16 that walk
// the prefix's positions together, RT tiles per work-group and the positions in
// `parts`; the sessions' own positions are walked as single tokens are, in
// pieces.  Both kinds of work-group are one launch, and the merge takes the
// parts and the pieces of a row.  Where that costs more than it saves, a session
// is one work-group's of k_window (attn_window.hip).
#include "attn_rows.h"

constexpr int SH_NW = 4;   // waves per work-group

// work-groups of the prefix: (kv head, part) fastest, padded to the eight XCDs,
// so the row blocks that read the same positions run on one XCD and its L2
__host__ __device__ inline unsigned shared_lanes(const RowsArgs &a) { return (unsigned)(a.n_kv * a.parts + 7) / 8 * 8; }
__host__ __device__ inline unsigned shared_prefix_wgs(const RowsArgs &a, int rt)
{
    const int rows = a.n * (a.n_heads / a.n_kv);
    return a.prefix ? shared_lanes(a) * (unsigned)((rows + 16 * rt - 1) / (16 * rt)) : 0;
}

template <int DH, typename KT, int RT>
__device__ __forceinline__ void shared_prefix(const RowsArgs &a, RowsMeet<DH, SH_NW> &meet, unsigned wg)
{
#pragma clang fp contract(off)
    const int G = a.n_heads / a.n_kv, rows = a.n * G;
    const unsigned lanes = shared_lanes(a), lane = wg % lanes;
    const int kvh = lane / a.parts, part = lane % a.parts, r0 = wg / lanes * 16 * RT;
    if (kvh >= a.n_kv) return;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    RowsLine<rw_tp<KT>()> line;
    line.s = line.lo = line.ns = 0;
    line.hi = a.prefix;
    const int T = line.tiles(), R = (T + a.parts - 1) / a.parts;
    const int u0 = min(part * R, T), u1 = min(u0 + R, T);
    RowsWave<DH, KT, RT> w;
    w.load([&](int r) {
        r = min(r0 + r, rows - 1);
        return a.q + ((size_t)(r / G) * a.n_heads + (size_t)kvh * G + r % G) * DH;
    });
    const size_t base = (size_t)kvh * a.prefix_ctx * DH;
    rows_walk<DH, KT, RT, false, false>(w, RowsFrom<KT>((const KT *)a.pk + base, (const KT *)a.pv + base), line, u0 + wid, u1, SH_NW,
                                 nullptr);
    const size_t x0 = ((size_t)kvh * rows + r0) * a.parts + part;
    rows_finish(w, meet, [&](int r, float m, float l, int d, auto &x) {
        if (r0 + r >= rows) return;
        const size_t at = x0 + (size_t)r * a.parts;
        rows_store(a.xo + at * DH + d, x);
        if (d == 0) {
            a.xm[at] = m;
            a.xl[at] = l;
        }
    });
}

template <int DH, typename KT, bool FEW, typename M>
__device__ __forceinline__ void shared_own(const RowsArgs &a, M &meet, unsigned wg)
{
#pragma clang fp contract(off)
    const int G = a.n_heads / a.n_kv, blocks = (G + 15) / 16;
    const int slot = wg / (a.n_kv * blocks), hb = wg % (a.n_kv * blocks), kvh = hb / blocks, r0 = hb % blocks * 16;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int TP = FEW ? FEW_TP : rw_tp<KT>();
    const RowsPiece p = rows_piece<TP>(a, slot);
    if (p.item < 0 || p.L <= 0) return;
    const RowsLine<TP> line = rows_line<TP>(p.L - 1, p.L - 1, a.window, a.sinks);
    const size_t row0 = (size_t)p.item * a.n_heads + (size_t)kvh * G;
    typename std::conditional<FEW, RowsFew<DH>, RowsWave<DH, KT, 1>>::type w;
    w.load([&](int r) { return a.q + (row0 + min(r0 + r, G - 1)) * DH; });
    const size_t base = (size_t)p.slot * a.slot_stride + (size_t)kvh * a.max_ctx * DH;
    const RowsFrom<KT> from((const KT *)a.k + base, (const KT *)a.v + base);
    if constexpr (FEW) few_walk<DH, false>(w, from, line, p.u0 + wid, p.u1, SH_NW);
    else rows_walk<DH, KT, 1, false, false>(w, from, line, p.u0 + wid, p.u1, SH_NW, nullptr);
    const size_t part = ((size_t)kvh * rows_slots(a) + slot) * G;
    auto put = [&](int r, float m, float l, int d, auto &x) {
        r += r0;
        if (r >= G) return;
        rows_store(a.po + (part + r) * DH + d, x);
        if (d == 0) {
            a.pm[part + r] = m;
            a.pl[part + r] = l;
        }
    };
    if constexpr (FEW) few_finish(w, meet, put);
    else rows_finish(w, meet, put);
}

// 48 sessions of 16/4 heads of 128 behind 2000 positions, fp32: 18.5 us, of which
// the prefix's f32 products are 6 at least; 32 sessions behind 8192, fp16, 56 MB:
// 19.3 us, most of it the start, the search for a piece and the end of work-groups
// with few steps.  The prefix's rows (columns of a product) are all used: n G of
// them share a tile of 16.
template <int DH, typename KT, int RT, bool FEW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DH == 256 ? 1 : 2))) void k_shared(RowsArgs a)
{
    __shared__ union {
        RowsMeet<DH, SH_NW> rows;
        FewMeet<DH, SH_NW> few;
    } meet;
    const unsigned pre = shared_prefix_wgs(a, RT);
    if (blockIdx.x < pre) shared_prefix<DH, KT, RT>(a, meet.rows, blockIdx.x);
    else if constexpr (FEW) shared_own<DH, KT, true>(a, meet.few, blockIdx.x - pre);
    else shared_own<DH, KT, false>(a, meet.rows, blockIdx.x - pre);
}

// One work-group per (query head, session): the prefix's parts and the session's
// pieces, 4.4 .. 5.3 us.
template <int DH, int TP>
__global__ __launch_bounds__(256) void k_shared_merge(RowsArgs a)
{
    constexpr int LPR = DH / 4;
    const int G = a.n_heads / a.n_kv, h = blockIdx.x, kvh = h / G, i = blockIdx.y, tid = threadIdx.x;
    const int pre = a.prefix ? a.parts : 0;
    int first;
    const int np = rows_pieces<TP>(a, i, &first);
    const size_t x0 = ((size_t)kvh * a.n * G + (size_t)i * G + h % G) * a.parts;
    const size_t p0 = ((size_t)kvh * rows_slots(a) + first) * G + h % G;
    const f32x4 o = rows_sum<DH, 256 / LPR, 4>(
        pre + np, tid % LPR, tid / LPR, [&](int j, const float **m, const float **l, const float **x) {
            const bool own = j >= pre;
            const size_t at = own ? p0 + (size_t)(j - pre) * G : x0 + j;
            *m = (own ? a.pm : a.xm) + at;
            *l = (own ? a.pl : a.xl) + at;
            *x = (own ? a.po : a.xo) + at * DH;
        });
    if (tid < LPR) *(f32x4 *)(a.out + ((size_t)i * a.n_heads + h) * DH + 4 * tid) = o;
}

// Row tiles of a prefix work-group: two over fp16 where there are rows for them
// and registers (a position read once for 32 rows), one over fp32, whose
// products take sixteen times as long and spread better in small pieces (48
// sessions of 4 heads behind 2000 positions: 22.1 against 23.2 us).
static int shared_rt(int n, int G, int d_head, int kv_f16)
{
    return (long)n * G <= 16 || d_head == 256 || !kv_f16 ? 1 : 2;
}

// Parts of the prefix.  Its work-groups and those of the own positions make one
// round of two per CU at 192 (32 sessions of 4 heads behind 8192 positions, fp16,
// in the kernel: 24.6 us at 96, 20.5 at 160, 21.2 at 192, 23.5 at 224, 26.4 at
// 512).  Where a wave then has more than twenty tiles to walk the prefix takes
// most of two per CU (65536 positions: 84 us at 192, 71 at 448; 16000 over fp32,
// 48 sessions: 103, 81; 320, which gives every fourth CU a second one, lies
// between).
constexpr int SH_WGS = 192;
static int shared_parts(int n, int n_heads, int n_kv, int prefix, int rt, int kv_f16)
{
    const long blocks = (long)n_kv * ceil_div((long)n * (n_heads / n_kv), 16 * rt);
    const long tiles = ceil_div(prefix, kv_f16 ? 32 : 16);
    const long wgs = tiles * blocks > 20L * SH_NW * SH_WGS ? 448 : SH_WGS;
    return (int)std::max(1L, std::min(wgs / blocks, (tiles + SH_NW - 1) / SH_NW));
}

// Whether every session is one work-group's (per kv head), prefix and own
// positions together: no merge launch, but the prefix read by each.  By what both
// are estimated to cost, in microseconds, from the most positions the call may
// have; apart: two launches, their pieces, the prefix's products (an f32 one as
// eight f16 ones) and the own positions' bytes.  Fitted to 2 .. 64 sessions of 16/4
// heads of 128 and 9/3 of 64 behind 100 .. 3200 positions with up to 100 .. 1500 of
// their own.  Both sides measured, apart and together: 8 sessions of 9/3 heads,
// fp16, 200 + 200: 8.9 and 5.6 us, 1600 + 128: 9.3 and 12.3; 64 of 16/4, fp16,
// 800 + 512: 22.2 and 17.2; 8 of 16/4, fp32, 200 + 200: 10.2 and 9.7, 800 + 128: 9.5
// and 15.4.
static bool shared_whole(int n, int n_heads, int n_kv, int d_head, int prefix, int max_ctx, int kv_f16)
{
    const int e = rows_whole_env();
    if (e >= 0) return e;
    const double wgs = (double)n * n_kv * ceil_div(n_heads / n_kv, 16);
    const double apart = 8.9 + 0.015 * n * n_kv + 5.1e-9 * n * n_heads * prefix * d_head * (kv_f16 ? 1 : 8) +
                         6.6e-8 * n * n_kv * max_ctx * d_head * (kv_f16 ? 4 : 8);
    return rows_together(wgs, (double)prefix + max_ctx, d_head, kv_f16) < apart;
}

RowsPlan rows_plan_shared(int n, int n_heads, int n_kv, int d_head, int prefix, int max_ctx)
{
    RowsPlan p;
    if (shared_whole(n, n_heads, n_kv, d_head, prefix, max_ctx, 0) && shared_whole(n, n_heads, n_kv, d_head, prefix, max_ctx, 1))
        return p;
    const int G = n_heads / n_kv;
    p.parts = 1;
    for (int f16 = 0; f16 < 2; f16++)
        p.parts = std::max(p.parts, shared_parts(n, n_heads, n_kv, prefix, shared_rt(n, G, d_head, f16), f16));
    p.cross = prefix ? (size_t)n * n_heads * p.parts : 0;
    // (own contexts of two tiles a wave at most: not cut; else pieces for what the
    // prefix leaves of two work-groups per CU: 32 sessions of 16/4 heads of 128 behind
    // 3000 positions, fp16, 21.8 us with pieces for all of them, 19.0)
    if (max_ctx > 8 * RW_PLAN_TP)
        p.bal = rows_plan_bal(n, (long)n_kv * ceil_div(G, 16), ceil_div(max_ctx, RW_PLAN_TP), RW_WGS - SH_WGS);
    p.pieces = (size_t)n_kv * (p.bal ? p.bal : n) * G;
    return p;
}

int launch_attn_shared(const RowsArgs &a0, hipStream_t s)
{
    RowsArgs a = a0;
    if (shared_whole(a.n, a.n_heads, a.n_kv, a.d_head, a.prefix, a.max_ctx, a.kv_f16)) {
        a.bal = 0;
        return launch_attn_window(a, s);
    }
    const int G = a.n_heads / a.n_kv, rt = shared_rt(a.n, G, a.d_head, a.kv_f16);
    a.parts = std::min(a.parts, shared_parts(a.n, a.n_heads, a.n_kv, a.prefix, rt, a.kv_f16));
    const dim3 grid(shared_prefix_wgs(a, rt) + (unsigned)(a.n_kv * ceil_div(G, 16)) * rows_slots(a)), block(256);
    const bool few = few_takes(a.d_head, G, a.kv_f16);
#define SHA(DH)                                                                                                  \
    if constexpr (few_takes(DH, 1, 0))                                                                           \
        if (few) hipLaunchKernelGGL((k_shared<DH, float, 1, true>), grid, block, 0, s, a);                       \
    if (!a.kv_f16 && !few) hipLaunchKernelGGL((k_shared<DH, float, 1, false>), grid, block, 0, s, a);            \
    if (a.kv_f16 && (DH == 256 || rt == 1)) hipLaunchKernelGGL((k_shared<DH, _Float16, 1, false>), grid, block, 0, s, a); \
    if (a.kv_f16 && rt == 2) hipLaunchKernelGGL((k_shared<DH, _Float16, DH == 256 ? 1 : 2, false>), grid, block, 0, s, a);
    RW_BY_D_HEAD(a.d_head, SHA)
#undef SHA
#define MERGE(DH)                                                                                     \
    if (a.kv_f16 || few) hipLaunchKernelGGL((k_shared_merge<DH, 32>), dim3(a.n_heads, a.n), block, 0, s, a); \
    else hipLaunchKernelGGL((k_shared_merge<DH, 16>), dim3(a.n_heads, a.n), block, 0, s, a);
    RW_BY_D_HEAD(a.d_head, MERGE)
#undef MERGE
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
