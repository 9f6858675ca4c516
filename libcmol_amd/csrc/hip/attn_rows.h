// attn_rows.h — attention of query rows whose visible positions are not simply
// the first seqlen of their own cache: a sliding window with sinks
// (attn_window.hip) and a prefix shared by the sessions (attn_shared.hip).
// An item is a session's token or a prompt token; query row (item, h) of kv
// head h / G sees
//   window   t <= p and (t < sinks or t > p - window), p = its position
//   shared   the prefix's positions, then its own t < seqlen
// and out = sum_t softmax_t(q . k_t / sqrt(d_head)) v_t over them, 0 where
// there are none.  Every sum and softmax statistic is fp32.
//
// One walk serves all of them (rows_walk): a wave holds RT tiles of 16 query
// rows of one kv head and takes tiles of TP cached positions (32 over fp16, 16
// over fp32: the same bytes), straight from the cache into the matrix
// instructions' operand registers; nothing is staged in LDS and the waves of a
// work-group, on different tiles, meet only at the end of their range
// (rows_finish).
//   * scores transposed, S^T = K Q^T: the A operand's rows are 16 positions
//     (16-byte pieces of the K rows as cached), the B operand's columns the
//     query rows, so lane (col, g) holds positions 4g .. 4g+3 of row `col` (of each
//     16);
//   * O^T += V^T P^T: the scores' layout is the B operand's as it is (k index
//     of lane group g = positions 4g .. 4g+3, and over fp16 those of the tile's
//     second 16), and a lane's A operand for output tile e is dimension
//     VD col + e of those positions, VD = d_head / 16: a lane loads VD neighbouring
//     dimensions of its positions' V rows, 16 lanes a whole row, and for fp16
//     pairs of rows are interleaved with one v_perm_b32 per two values;
//   * online softmax whose reference moves only when a score exceeds it by more
//     than RW_LAZY (log2 units; a wave vote), so most tiles need no cross-lane
//     step; weights are 2^(t c2 + mk), c2 = log2(e) / sqrt(d_head).
// fp16 caches: 16x16x32 f16 products, exact, with fp32 sums.  The query is
// scaled by a power of two per row into [2^9, 2^10) and split into two f16 parts
// (22 bits, 2^-33 of the row's largest below) whose products share a sum; a
// weight, scaled by 2^RW_SCALE, into two f16 parts whose products share an
// accumulator (22 bits of a weight down to 2^-16 of the largest, an absolute
// 2^-36 of it below).  fp32 caches: 16x16x4 f32 products throughout; a few rows
// by themselves have a walk of their own (few_walk).
#pragma once
#include "lanes.h"

#include <algorithm>
#include <utility>

template <typename KT> constexpr int rw_tp() { return sizeof(KT) == 2 ? 32 : 16; }   // positions per tile
constexpr float RW_LAZY = 2.0f;      // log2: weights stay below 2^(RW_SCALE + 2)
constexpr float RW_SCALE = 12.0f;

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
    // work split (rows_plan_*) and its partial results: (m, l, o[d_head]) per
    // query row and part; a weight sum is l 2^m
    int bal;                   // pieces of the items' own positions at most (0: one work-group per item)
    int parts;                 // parts of the prefix, or of a prompt block's positions
    float *pm, *pl, *po;       // [n_kv][rows_slots][G]
    float *xm, *xl, *xo;       // [n_kv][n * G][parts]
    void *split;               // prompt over an fp32 cache: its f16 pairs (attn_wprompt.hip)
};

// ---- which positions -----------------------------------------------------------

// Tiles of two runs of positions, [0, s) and [lo, hi): the first ns tiles
// cover the first, the rest the second (of another cache, where the first is a
// shared prefix).
template <int TP>
struct RowsLine {
    int s, lo, hi, ns;
    __device__ __forceinline__ int tiles() const { return ns + (hi - lo + TP - 1) / TP; }
    // first position and number of positions of tile u
    __device__ __forceinline__ void tile(int u, int *p0, int *cnt) const
    {
        *p0 = u < ns ? u * TP : lo + (u - ns) * TP;
        *cnt = min(TP, (u < ns ? s : hi) - *p0);
    }
    // in scalar registers: what follows from them is too, and branches on it are
    // scalar ones (the lines and ranges of a wave are uniform, which the compiler
    // cannot see through the search of a piece)
    __device__ __forceinline__ RowsLine uniform() const
    {
        RowsLine x;
        x.s = __builtin_amdgcn_readfirstlane(s);
        x.lo = __builtin_amdgcn_readfirstlane(lo);
        x.hi = __builtin_amdgcn_readfirstlane(hi);
        x.ns = __builtin_amdgcn_readfirstlane(ns);
        return x;
    }
};

// Positions that tokens at first .. last see between them.
template <int TP>
__device__ __forceinline__ RowsLine<TP> rows_line(int first, int last, int window, int sinks)
{
    RowsLine<TP> l;
    l.hi = last + 1;
    l.lo = max(first + 1 - window, 0);
    l.s = min(sinks, l.lo);
    l.ns = (l.s + TP - 1) / TP;
    return l;
}

// Item i: positions of its cache up to its own (0: it sees nothing there), and
// which cache.
__device__ __forceinline__ int rows_item(const RowsArgs &a, int i, int *slot)
{
    const int L = a.seqlen[i];
    *slot = a.slots ? a.slots[i] : i;
    return *slot < 0 ? 0 : max(min(L, a.max_ctx), 0);
}

template <int TP>
__device__ __forceinline__ unsigned rows_tiles(const RowsArgs &a, int L)
{
    return L > 0 ? rows_line<TP>(L - 1, L - 1, a.window, a.sinks).tiles() : 0;
}

// Pieces.  The items are cut into pieces of at most R tiles, each into equal ones
// as far as they go, with R the least at which there are no more pieces than
// `bal` work-groups; slot k holds the k-th piece in the items' order, so an item's
// are consecutive, and every work-group finds its own, if any, from the lengths
// alone.  (Ranges of one line of all tiles cut the items anywhere: 64 sessions of
// 16/4 heads, windows of 2000, fp16: 64 us.)
constexpr unsigned RW_RMIN = 4;   // tiles per piece to have, one per wave

__host__ __device__ inline int rows_slots(const RowsArgs &a) { return a.bal ? a.bal : a.n; }

// a / b; `small`: a below 2^21, where half a unit more, times the hardware
// reciprocal, is off by less than that half (an integer division is a chain of 25
// instructions).
__device__ __forceinline__ unsigned rows_div(unsigned a, unsigned b, bool small)
{
    return small ? (unsigned)(((float)a + 0.5f) * __builtin_amdgcn_rcpf((float)b)) : a / b;
}

// A lane's item among the first 64, and the most tiles of a piece (every wave
// works them out, with no barrier).
template <int TP>
struct RowsSpread {
    int L, slot;
    unsigned T, R, V;   // its tiles; the most of a piece; its pieces
    bool small;   // T and R below 2^20
    __device__ __forceinline__ explicit RowsSpread(const RowsArgs &a)
    {
        const int lane = threadIdx.x & 63;
        item(a, lane);
        small = a.max_ctx < 1 << 23;
        if (a.n <= 64) {
            R = RW_RMIN;
            V = (T + RW_RMIN - 1) / RW_RMIN;
            if (wave_sum_u(V) > (unsigned)a.bal) {
                // (at twice the least there are at most bal / 2 + n, and bal >= 2 n)
                const unsigned t = wave_sum_u(T);
                const unsigned r = max(RW_RMIN, small ? (unsigned)((float)t * __builtin_amdgcn_rcpf((float)a.bal)) + 1 : t / a.bal + 1);
                for (unsigned k = 0; k <= 8; k++) {
                    R = r + r * k / 8;
                    V = pieces(T);
                    if (wave_sum_u(V) <= (unsigned)a.bal) break;
                }
            }
        } else {   // (at most bal - n, and one more an item)
            unsigned t = T;
            for (int b = 64; b < a.n; b += 64) {
                int s;
                if (b + lane < a.n) t += rows_tiles<TP>(a, rows_item(a, b + lane, &s));
            }
            R = max(RW_RMIN, (wave_sum_u(t) + a.bal - a.n - 1) / (a.bal - a.n));
            V = pieces(T);
        }
    }
    __device__ __forceinline__ unsigned pieces(unsigned tiles) const { return rows_div(tiles + R - 1, R, small); }
    __device__ __forceinline__ void item(const RowsArgs &a, int i)
    {
        slot = -1;
        L = i < a.n ? rows_item(a, i, &slot) : 0;
        T = rows_tiles<TP>(a, L);
    }
};

struct RowsPiece {
    int item, L, slot, u0, u1;   // item below 0: no piece
    bool whole;                  // the item's only one
};
// The piece of work-group slot k, or item k whole where there are no pieces.
template <int TP>
__device__ __forceinline__ RowsPiece rows_piece(const RowsArgs &a, int k)
{
    RowsPiece p;
    if (!a.bal) {
        p.item = k;
        p.L = rows_item(a, k, &p.slot);
        p.u0 = 0;
        p.u1 = rows_tiles<TP>(a, p.L);
        p.whole = true;
        return p;
    }
    const int lane = threadIdx.x & 63;
    RowsSpread<TP> x(a);
    unsigned base = 0;
    p.item = -1;
    for (int b = 0; b < a.n; b += 64) {
        if (b) {
            x.item(a, b + lane);
            x.V = x.pieces(x.T);
        }
        const unsigned v = x.V, inc = wave_scan_u(v), at = base + inc - v;
        const uint64_t m = __ballot((unsigned)k - at < v);
        if (m) {
            const int j = __builtin_ctzll(m);
            const unsigned n = __builtin_amdgcn_readlane(v, j), q = k - __builtin_amdgcn_readlane(at, j);
            const unsigned T = __builtin_amdgcn_readlane(x.T, j), each = rows_div(T, n, x.small), more = T - each * n;
            p.item = b + j;
            p.L = __builtin_amdgcn_readlane(x.L, j);
            p.slot = __builtin_amdgcn_readlane(x.slot, j);
            p.u0 = q * each + min(q, more);
            p.u1 = p.u0 + each + (q < more);
            p.whole = n == 1;
            break;
        }
        base += __builtin_amdgcn_readlane(inc, 63);
    }
    return p;
}

// The slots of item i's pieces: the first, and how many.
template <int TP>
__device__ __forceinline__ int rows_pieces(const RowsArgs &a, int i, int *first)
{
    int slot;
    if (!a.bal) {
        *first = i;
        return rows_item(a, i, &slot) > 0 ? 1 : 0;
    }
    const int lane = threadIdx.x & 63;
    const RowsSpread<TP> x(a);
    unsigned pre = lane < min(i, 64) ? x.V : 0;
    for (int b = 64; b < i; b += 64)
        if (b + lane < i) pre += x.pieces(rows_tiles<TP>(a, rows_item(a, b + lane, &slot)));
    *first = wave_sum_u(pre);
    return i < 64 ? __builtin_amdgcn_readlane(x.V, i) : x.pieces(rows_tiles<TP>(a, rows_item(a, i, &slot)));
}

// ---- the walk ------------------------------------------------------------------

// A wave's query rows and their online softmaxes: lane (col, g) = (lane % 16,
// lane / 16) holds row 16 rt + col of tile rt.
template <int DH, typename KT, int RT>
struct RowsWave {
    static constexpr bool F16 = sizeof(KT) == 2;
    static constexpr int VD = DH / 16;               // dimensions per lane of a V row, output tiles
    static constexpr int KS = DH < 32 ? 1 : DH / 32; // f16 k-steps of a score
    f16x8 qh[RT][F16 ? KS : 1], ql[RT][F16 ? KS : 1];
    f32x4 qf[RT][F16 ? 1 : VD];
    float c2[RT];            // log2 units per raw score
    f32x4 o[RT][VD];         // o[rt][e][i]: dimension VD (4g + i) + e of the row
    float m[RT], mk[RT], l[RT];   // l: this lane's positions only

    // Row r's query at q(r): loaded first, made an operand once the first cached
    // rows are on their way.
    static constexpr int XR = F16 ? KS * 8 : VD * 4;
    float x[RT][XR];
    template <typename Q>
    __device__ __forceinline__ void load(Q q)
    {
        const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float *p = q(16 * rt + col);
#pragma unroll
            for (int i = 0; i < XR / 4; i++) {
                const f32x4 y = F16 ? ldg((const f32x4 *)(p + (32 * (i / 2) + 8 * g) % DH + 4 * (i & 1)))
                                    : ldg((const f32x4 *)(p + 16 * i + 4 * g));
#pragma unroll
                for (int e = 0; e < 4; e++) x[rt][4 * i + e] = y[e];
            }
        }
    }
    __device__ __forceinline__ void convert()
    {
#pragma clang fp contract(off)
        const int g = (threadIdx.x & 63) >> 4;
        const float sc = 1.44269504088896341f / sqrtf((float)DH);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            c2[rt] = sc;
            if constexpr (F16) {
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < XR; i++) {
                    if (DH < 32 && g >= 2) x[rt][i] = 0.0f;   // (d_head 16: half a k-step)
                    top = fmaxf(top, fabsf(x[rt][i]));
                }
                top = lanes_max<32>(lanes_max<16>(top));
                // the largest into [2^9, 2^10), so that the low parts are normal
                // numbers too (below 2^-100 less, so that c2 stays above 0); a row
                // of zeros, infinities or NaN as it is
                const int ex = top > 0.0f && top < INFINITY ? max(__builtin_amdgcn_frexp_expf(top) - 1, -100) - 9 : 0;
                c2[rt] = ldexpf(sc, ex);
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float y = __builtin_amdgcn_ldexpf(x[rt][8 * s + e], -ex);
                        const _Float16 hi = (_Float16)y;
                        qh[rt][s][e] = hi;
                        ql[rt][s][e] = (_Float16)(y - (float)hi);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < VD; i++) qf[rt][i] = f32x4{x[rt][4 * i], x[rt][4 * i + 1], x[rt][4 * i + 2], x[rt][4 * i + 3]};
            }
            m[rt] = -INFINITY;
            mk[rt] = RW_SCALE;
            l[rt] = 0.0f;
#pragma unroll
            for (int e = 0; e < VD; e++) o[rt][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
};

// Mask of the rows of a prompt block: row r's token is at position pos[rt].
struct RowsSeen {
    int first, last, window, sinks;   // positions of the block's tokens
    const int *pos;
};

// K and V rows of the kv head: the first run's, the second's.
template <typename KT>
struct RowsFrom {
    const KT *k1, *v1, *k, *v;
    __device__ __forceinline__ RowsFrom(const KT *k0, const KT *v0) : k1(k0), v1(v0), k(k0), v(v0) {}
    __device__ __forceinline__ RowsFrom(const KT *pk, const KT *pv, const KT *k0, const KT *v0) : k1(pk), v1(pv), k(k0), v(v0) {}
};

// A 16-byte load; NT: of what the call reads once.
template <bool NT, typename T>
__device__ __forceinline__ T rows_ldg(const T *p)
{
    static_assert(sizeof(T) == 16, "16 bytes");
    if constexpr (NT) return __builtin_nontemporal_load(gptr(p));
    else return ldg(p);
}

// Tiles u, u + step, .. below u1 of `line` into the wave's rows (loaded, not yet
// converted).  MASKED: rows see different positions (seen).
template <int DH, typename KT, int RT, bool MASKED, bool NT>
__device__ __forceinline__ void rows_walk(RowsWave<DH, KT, RT> &w, const RowsFrom<KT> &from,
                                          const RowsLine<rw_tp<KT>()> &line0, int u, int u1, int step, const RowsSeen *seen)
{
#pragma clang fp contract(off)
    const auto line = line0.uniform();
    u = __builtin_amdgcn_readfirstlane(u);
    u1 = __builtin_amdgcn_readfirstlane(u1);
    typedef RowsWave<DH, KT, RT> W;
    constexpr bool F16 = W::F16;
    constexpr int VD = W::VD, KS = W::KS, ES = sizeof(KT), TP = rw_tp<KT>(), C = TP / 16, VR = TP / 4;
    constexpr int VB = VD * ES;                        // bytes of a lane's piece of a V row
    constexpr int VW = VB < 4 ? 1 : VB / 4;            // dwords of it
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const f32x4 zero4 = {0.0f, 0.0f, 0.0f, 0.0f};
    f16x8 kh[F16 ? C : 1][F16 ? KS : 1];
    f32x4 kf[F16 ? 1 : VD];
    uint32_t vr[VR][VW];                               // V rows 16 (r / 4) + 4g + r % 4
    auto load_k = [&](int t) {
        int p0, cnt;
        line.tile(t, &p0, &cnt);
        const char *base = (const char *)uniform_ptr((t < line.ns ? from.k1 : from.k) + (size_t)p0 * DH);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const unsigned at = (unsigned)min(16 * c + col, cnt - 1) * (DH * ES);
            if constexpr (F16) {
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    kh[c][s] = rows_ldg<NT>((const f16x8 *)(base + (at + (64 * s + 16 * g) % (DH * ES))));
                    if (DH < 32 && g >= 2) kh[c][s] = f16x8{};
                }
            } else {
#pragma unroll
                for (int i = 0; i < VD; i++) kf[i] = rows_ldg<NT>((const f32x4 *)(base + (at + 64 * i + 16 * g)));
            }
        }
    };
    auto load_v = [&](int t) {
        int p0, cnt;
        line.tile(t, &p0, &cnt);
        const char *base = (const char *)uniform_ptr((t < line.ns ? from.v1 : from.v) + (size_t)p0 * DH);
#pragma unroll
        for (int r = 0; r < VR; r++) {
            const int row = 16 * (r / 4) + 4 * g + r % 4;
            const char *src = base + ((unsigned)min(row, cnt - 1) * (DH * ES) + VB * col);
            if constexpr (VB == 2) vr[r][0] = *gptr((const uint16_t *)src);
            else if constexpr (VB == 4) vr[r][0] = ldg((const uint32_t *)src);
            else if constexpr (VB == 8) {
                const u32x2 x = ldg((const u32x2 *)src);
                vr[r][0] = x[0];
                vr[r][1] = x[1];
            } else {
#pragma unroll
                for (int b = 0; b < VB / 16; b++) {
                    const u32x4 x = rows_ldg<NT>((const u32x4 *)(src + 16 * b));
#pragma unroll
                    for (int e = 0; e < 4; e++) vr[r][4 * b + e] = x[e];
                }
            }
        }
    };
    if (u < u1) {
        load_k(u);
        load_v(u);
    }
    w.convert();
    for (; u < u1; u += step) {
        int p0, cnt;
        line.tile(u, &p0, &cnt);
        // ---- scores: sc[rt][c][i] = position p0 + 16c + 4g + i of row 16 rt + col
        f32x4 sc[RT][C];
#pragma unroll
        for (int c = 0; c < C; c++) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                sc[rt][c] = zero4;
                if constexpr (F16) {
#pragma unroll
                    for (int s = 0; s < KS; s++) {
                        sc[rt][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[c][s], w.ql[rt][s], sc[rt][c], 0, 0, 0);
                        sc[rt][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[c][s], w.qh[rt][s], sc[rt][c], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int d = 0; d < VD; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            sc[rt][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[d][e], w.qf[rt][d][e], sc[rt][c], 0, 0, 0);
                }
            }
        }
        if (u + step < u1) load_k(u + step);
        // ---- masks (uniform branches): the run's end; rows that see less
        bool edge = cnt < TP;
        if constexpr (MASKED)
            edge |= p0 + cnt - 1 > seen->first || (p0 + cnt - 1 >= seen->sinks && p0 <= seen->last - seen->window);
        if (edge) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int at = 16 * c + 4 * g + i, p = p0 + at;
                        bool see = at < cnt;
                        if constexpr (MASKED)
                            see = see && p <= seen->pos[rt] && (p < seen->sinks || p > seen->pos[rt] - seen->window);
                        if (!see) sc[rt][c][i] = -INFINITY;
                    }
        }
        // V rows past the run: 0, not a copy of its last (0 weight times infinity)
        if (cnt < TP) {
#pragma unroll
            for (int r = 0; r < VR; r++)
                if (16 * (r / 4) + 4 * g + r % 4 >= cnt) {
#pragma unroll
                    for (int e = 0; e < VW; e++) vr[r][e] = 0;
                }
        }
        // ---- online softmax
        float mx[RT];
        bool up = false;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            mx[rt] = sc[rt][0][0];
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx[rt] = fmaxf(mx[rt], sc[rt][c][i]);
            up |= (mx[rt] - w.m[rt]) * w.c2[rt] > RW_LAZY;
        }
        if (__ballot(up)) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                mx[rt] = lanes_max<32>(lanes_max<16>(mx[rt]));
                const float mn = fmaxf(w.m[rt], mx[rt]);
                const float mkn = mn == -INFINITY ? RW_SCALE : RW_SCALE - mn * w.c2[rt];
                const float al = w.m[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mkn - w.mk[rt]);
                w.m[rt] = mn;
                w.mk[rt] = mkn;
                w.l[rt] *= al;
#pragma unroll
                for (int e = 0; e < VD; e++) w.o[rt][e] *= al;
            }
        }
        f16x8 ph[F16 ? RT : 1], pl[F16 ? RT : 1];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float ls = 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[rt][c][i], w.c2[rt], w.mk[rt]));
                    const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[rt][c][i + 1], w.c2[rt], w.mk[rt]));
                    ls += e0 + e1;
                    if constexpr (F16) {
                        const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(e0, e1));
                        const f16x2 lo = __builtin_bit_cast(
                            f16x2, __builtin_amdgcn_cvt_pkrtz(e0 - (float)hi[0], e1 - (float)hi[1]));
                        ph[rt][4 * c + i] = hi[0];
                        ph[rt][4 * c + i + 1] = hi[1];
                        pl[rt][4 * c + i] = lo[0];
                        pl[rt][4 * c + i + 1] = lo[1];
                    } else {
                        sc[rt][c][i] = e0;
                        sc[rt][c][i + 1] = e1;
                    }
                }
            w.l[rt] += ls;
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int e = 0; e < VD; e++) {
            if constexpr (F16) {
                u32x4 x;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    x[j] = __builtin_amdgcn_perm(vr[2 * j + 1][e / 2], vr[2 * j][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
                const f16x8 va = __builtin_bit_cast(f16x8, x);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) w.o[rt][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[rt], w.o[rt][e], 0, 0, 0);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) w.o[rt][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[rt], w.o[rt][e], 0, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
                        w.o[rt][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[j][e]), sc[rt][0][j], w.o[rt][e], 0, 0, 0);
            }
        }
        if (u + step < u1) load_v(u + step);
    }
}

// The waves of a work-group meet: put(r, m, l, d, x) gets, for every row r of
// the work-group's 16 RT, its sums over the waves: weight sum l 2^m and
// the unnormalised output's dimensions d .. d+N-1 (x), from one thread each.
template <int DH, int NW>
struct RowsMeet {
    static constexpr int DC = DH < 512 / NW ? DH : 512 / NW;   // dimensions per round (34 KiB)
    __attribute__((aligned(16))) float o[NW][16][DC + 4];
    float m[NW][16], l[NW][16];
};
template <int DH, typename KT, int RT, int NW, typename P>
__device__ __forceinline__ void rows_finish(RowsWave<DH, KT, RT> &w, RowsMeet<DH, NW> &meet, P put)
{
#pragma clang fp contract(off)
    constexpr int VD = DH / 16, DC = RowsMeet<DH, NW>::DC, TPR = NW * 4;   // threads per row
    constexpr int N = DC / TPR < 1 ? 1 : DC / TPR;                        // dimensions per thread and round
    auto &xo = meet.o;
    auto &xm = meet.m, &xl = meet.l;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, col = lane & 15, g = lane >> 4;
    const int r = tid / TPR, a = tid % TPR;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const float l = lanes_add<32>(lanes_add<16>(w.l[rt]));
        // a lane's dimensions VD (4g + i) .. +VD-1 of round c: those in [c DC, c DC + DC)
#pragma unroll
        for (int c = 0; c < DH / DC; c++) {
            if (rt || c) __syncthreads();
            if (g == 0 && c == 0) {
                xm[wid][col] = w.m[rt] == -INFINITY ? -INFINITY : -w.mk[rt];
                xl[wid][col] = l;
            }
            if (VD * 4 * g / DC == c) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < VD; e++) xo[wid][col][VD * (4 * g + i) - c * DC + e] = w.o[rt][e][i];
            }
            __syncthreads();
            float mx = xm[0][r];
#pragma unroll
            for (int k = 1; k < NW; k++) mx = fmaxf(mx, xm[k][r]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float lt = 0.0f, x[N] = {};
            const bool on = N * a < DC;   // (d_head 16 over eight waves: half of the threads)
#pragma unroll
            for (int k = 0; k < NW; k++) {
                const float f = __builtin_amdgcn_exp2f(xm[k][r] - ref);
                lt += xl[k][r] * f;
#pragma unroll
                for (int e = 0; e < N; e++) x[e] += on ? xo[k][r][N * a + e] * f : 0.0f;
            }
            if (on) put(16 * rt + r, mx, lt, c * DC + N * a, x);
        }
    }
}

template <int N>
__device__ __forceinline__ void rows_store(float *p, const float (&x)[N])
{
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int e = 0; e < N; e += 4) *(f32x4 *)(p + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) p[e] = x[e];
    }
}

// ---- few rows over fp32 ----------------------------------------------------------
// At most four query rows of a kv head (its group, for single tokens) over an
// fp32 cache at d_head 64 and 128.  Of the 16 columns of a 16x16x4 f32 product
// they would use four; 4x4x1 f32 products, 16 blocks an instruction, run at the
// same rate and waste none.  Tiles of 32 positions:
//   * a cached row is GL = d_head / 4 lanes of 16 bytes, an instruction loads NQ =
//     64 / GL whole rows: load n of a tile rows NQ n + q, q = lane / GL;
//   * scores: the quads' lanes hold dimensions, the products want positions: four
//     loads' registers are transposed within the quads (two DPP exchanges), lane t
//     then holds position 4i + t of the loads (A) against the four rows (B) over
//     16 dimensions of its block.  The sums over the blocks of a row are
//     reduce-scattered (lane swaps of 16, DPP for 8 and 4): lane 4b + h ends
//     with two positions of row h, those of V loads 2 (b % (GL / 4)) + 0 and 1;
//   * that is the A operand of the second product, whose blocks of a V row's
//     lanes share one position: the broadcast takes it from one block of each
//     group of GL / 4.
// Bound by the cache's bytes on their way into the CUs.  16 sessions of 15/5 heads
// of 64, windows of 601: 9.95 us by 16x16x4 products, 8.0 by these; 100 sessions
// 21.1, 19.8; 64 of windows of 2000 66, 62; 48 sessions' own positions behind a
// prefix (d_head 128) 21.7, 18.9 in the kernel; one session's window of 128 alike.
constexpr int FEW_ROWS = 4, FEW_TP = 32;
constexpr bool few_takes(int d_head, int group, int kv_f16)
{
    return !kv_f16 && group <= FEW_ROWS && (d_head == 64 || d_head == 128);
}

template <int DH, int NW>
struct FewMeet {
    __attribute__((aligned(16))) float o[NW][FEW_ROWS][DH];
    float m[NW][FEW_ROWS], l[NW][FEW_ROWS];
};

template <int DH>
struct RowsFew {
    static constexpr int GL = DH / 4, NQ = 64 / GL, NV = FEW_TP / NQ;
    f32x4 q[4];     // q[t][e]: dimension 16 (b % (GL / 4)) + 4t + e of row h
    f32x4 o[4];     // o[e][h]: dimension 4 (lane % GL) + e of row h, the positions of group lane / GL
    float m, mk, l; // of row h; l: this lane's positions only
    template <typename Q>
    __device__ __forceinline__ void load(Q at)
    {
        const int lane = threadIdx.x & 63;
        const float *p = at(lane & 3) + 16 * (lane % GL / 4);
#pragma unroll
        for (int t = 0; t < 4; t++) q[t] = ldg((const f32x4 *)(p + 4 * t));
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m = -INFINITY;
        mk = RW_SCALE;
        l = 0.0f;
    }
    // V rows n of every group, the weights of block n / 2 of each
    template <int... N>
    __device__ __forceinline__ void add(const f32x4 (&v)[NV], const float (&p)[2], std::integer_sequence<int, N...>)
    {
        (add_one<N>(v[N], p[N & 1]), ...);
    }
    template <int N>
    __device__ __forceinline__ void add_one(f32x4 v, float p)
    {
        // (one value of four registers up to here: the compiler gave a lane of it
        // away to the weights' arithmetic, before its product)
        asm volatile("" : "+v"(v));
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = __builtin_amdgcn_mfma_f32_4x4x1f32(p, v[e], o[e], GL == 16 ? 2 : 3, N >> 1, 0);
    }
};

// Two registers' transposition with the lane O away: the lower one's (on
// false) second against the upper one's first.
template <int O>
__device__ __forceinline__ void few_exchange(bool on, float a, float b, float &x, float &y)
{
    const float fa = lane_xor<O>(a), fb = lane_xor<O>(b);
    x = on ? fb : a;
    y = on ? b : fa;
}

// As rows_walk: tiles u, u + step, .. below u1.
template <int DH, bool NT>
__device__ __forceinline__ void few_walk(RowsFew<DH> &w, const RowsFrom<float> &from, const RowsLine<FEW_TP> &line0, int u,
                                         int u1, int step)
{
#pragma clang fp contract(off)
    const auto line = line0.uniform();
    u = __builtin_amdgcn_readfirstlane(u);
    u1 = __builtin_amdgcn_readfirstlane(u1);
    typedef RowsFew<DH> W;
    constexpr int TP = FEW_TP, GL = W::GL, NQ = W::NQ, NV = W::NV, NJ = NV / 4;
    const int lane = threadIdx.x & 63, b = lane >> 2, q = lane / GL;
    const float c2 = 1.44269504088896341f / sqrtf((float)DH);
    f32x4 kr[NV], vr[NV];
    auto load = [&](const float *run1, const float *run2, int t, f32x4 (&to)[NV]) {
        int p0, cnt;
        line.tile(t, &p0, &cnt);
        const char *base = (const char *)uniform_ptr((t < line.ns ? run1 : run2) + (size_t)p0 * DH);
#pragma unroll
        for (int n = 0; n < NV; n++)
            to[n] = rows_ldg<NT>((const f32x4 *)(base + ((unsigned)min(NQ * n + q, cnt - 1) * (DH * 4) + 16 * (lane % GL))));
    };
    if (u >= u1) return;
    load(from.k1, from.k, u, kr);
    load(from.v1, from.v, u, vr);
    for (;;) {
        const bool more = u + step < u1;
        int p0, cnt;
        line.tile(u, &p0, &cnt);
        f32x4 s[NJ];
#pragma unroll
        for (int j = 0; j < NJ; j++) s[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const bool l1 = lane & 1, l2 = lane & 2;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float z[NJ][4];
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const float r0 = kr[4 * j][e], r1 = kr[4 * j + 1][e], r2 = kr[4 * j + 2][e], r3 = kr[4 * j + 3][e];
                float y0, y1, y2, y3;
                few_exchange<1>(l1, r0, r1, y0, y1);
                few_exchange<1>(l1, r2, r3, y2, y3);
                few_exchange<2>(l2, y0, y2, z[j][0], z[j][2]);
                few_exchange<2>(l2, y1, y3, z[j][1], z[j][3]);
            }
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int j = 0; j < NJ; j++) s[j] = __builtin_amdgcn_mfma_f32_4x4x1f32(z[j][t], w.q[t][e], s[j], 0, 0, 0);
        }
        if (more) load(from.k1, from.k, u + step, kr);
        // ---- reduce-scatter: x[4j + i] is row NQ (4j + i) + q of the tile
        float x[NV], p[2];
#pragma unroll
        for (int i = 0; i < NV; i++) x[i] = s[i / 4][i % 4];
        if constexpr (GL == 32) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[i]), __float_as_uint(x[i + 8]), false, false);
                x[i] = __uint_as_float(y[0]) + __uint_as_float(y[1]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool on = lane & 8;
            x[i] = (on ? x[i + 4] : x[i]) + lane_xor<8>(on ? x[i] : x[i + 4]);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const bool on = lane & 4;
            p[i] = (on ? x[i + 2] : x[i]) + lane_xor<4>(on ? x[i] : x[i + 2]);
        }
        // ---- the run's end: V rows past it 0, not a copy of its last (0 weight times infinity)
        if (cnt < TP) {
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (NQ * (2 * (b % (GL / 4)) + i) + q >= cnt) p[i] = -INFINITY;
#pragma unroll
            for (int n = 0; n < NV; n++)
                if (NQ * n + q >= cnt) vr[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        // ---- online softmax
        float mx = fmaxf(p[0], p[1]);
        if (__ballot((mx - w.m) * c2 > RW_LAZY)) {
            mx = lanes_max<32>(lanes_max<16>(lanes_max<8>(lanes_max<4>(mx))));
            const float mn = fmaxf(w.m, mx), mkn = mn == -INFINITY ? RW_SCALE : RW_SCALE - mn * c2;
            const float al = w.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mkn - w.mk);
            w.m = mn;
            w.mk = mkn;
            w.l *= al;
#pragma unroll
            for (int h = 0; h < FEW_ROWS; h++) {
                const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(al), h));
#pragma unroll
                for (int e = 0; e < 4; e++) w.o[e][h] *= f;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], c2, w.mk));
            w.l += p[i];
        }
        w.add(vr, p, std::make_integer_sequence<int, NV>());
        if (!more) return;
        u += step;
        load(from.v1, from.v, u, vr);
    }
}

// As rows_finish, put(r, m, l, d, x) for rows below FEW_ROWS.
template <int DH, int NW, typename P>
__device__ __forceinline__ void few_finish(RowsFew<DH> &w, FewMeet<DH, NW> &meet, P put)
{
#pragma clang fp contract(off)
    constexpr int GL = RowsFew<DH>::GL;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const float l = lanes_add<32>(lanes_add<16>(lanes_add<8>(lanes_add<4>(w.l))));
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
        for (int h = 0; h < FEW_ROWS; h++) w.o[e][h] = lanes_add<32>(GL == 16 ? lanes_add<16>(w.o[e][h]) : w.o[e][h]);
    if (lane < FEW_ROWS) {
        meet.m[wid][lane] = w.m == -INFINITY ? -INFINITY : -w.mk;
        meet.l[wid][lane] = l;
    }
    if (lane < GL) {
#pragma unroll
        for (int h = 0; h < FEW_ROWS; h++)
            *(f32x4 *)&meet.o[wid][h][4 * lane] = f32x4{w.o[0][h], w.o[1][h], w.o[2][h], w.o[3][h]};
    }
    __syncthreads();
    if (tid >= FEW_ROWS * GL) return;
    const int r = tid / GL, d = 4 * (tid % GL);
    float mx = meet.m[0][r];
#pragma unroll
    for (int k = 1; k < NW; k++) mx = fmaxf(mx, meet.m[k][r]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float lt = 0.0f, x[4] = {};
#pragma unroll
    for (int k = 0; k < NW; k++) {
        const float f = __builtin_amdgcn_exp2f(meet.m[k][r] - ref);
        lt += meet.l[k][r] * f;
        const f32x4 y = *(const f32x4 *)&meet.o[k][r][d];
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += y[e] * f;
    }
    put(r, mx, lt, d, x);
}

// ---- one row on one wave ---------------------------------------------------------
// Lane l holds dimensions DL l .. +DL-1 (the first d_head lanes below 64).
template <int DH>
struct RowState {
    static constexpr int DL = DH < 64 ? 1 : DH / 64;
    float q[DL], o[DL], m, l;   // m in log2 units
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
    const float sc = 1.44269504088896341f / sqrtf((float)DH);
    for (int t = t0; t < t1; t++) {
        const size_t at = (size_t)t * DH + (on ? lane * DL : 0);
        float s = 0.0f;
#pragma unroll
        for (int d = 0; d < DL; d++) s = fmaf(r.q[d], (float)k[at + d], s);
        s = wave_sum(on ? s : 0.0f) * sc;
        const float mn = fmaxf(r.m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float al = exp2f(r.m - ref), e = exp2f(s - ref);
        r.m = s != s ? s : mn;   // (fmaxf drops a NaN)
        r.l = r.l * al + e;
#pragma unroll
        for (int d = 0; d < DL; d++) r.o[d] = r.o[d] * al + e * (float)v[at + d];
    }
}

// ---- partial results -------------------------------------------------------------

// The sum of a row's partial results by the LPR SG threads (d4, sg) of it, SG
// groups taking every SG-th, U at a time; at(j): where the j-th of np is.  Group
// 0's threads get the finished dimensions 4 d4 .. +3 (np 0: zeros).
template <int DH, int SG, int U, typename F>
__device__ __forceinline__ f32x4 rows_sum(int np, int d4, int sg, F at)
{
#pragma clang fp contract(off)
    float mx = -INFINITY, L = 0.0f;
    f32x4 acc = {};
    for (int j0 = sg; j0 < np; j0 += U * SG) {
        float pm[U], pl[U];
        f32x4 po[U];
#pragma unroll
        for (int i = 0; i < U; i++) {
            pm[i] = -INFINITY;
            if (SG == 1 && j0 + i >= np) continue;   // (uniform)
            const float *m, *l, *o;
            at(min(j0 + i * SG, np - 1), &m, &l, &o);
            pm[i] = j0 + i * SG < np ? *m : -INFINITY;
            pl[i] = *l;
            po[i] = *(const f32x4 *)(o + 4 * d4);
        }
        float mn = mx;
#pragma unroll
        for (int i = 0; i < U; i++) mn = fmaxf(mn, pm[i]);
        const float ref = mn == -INFINITY ? 0.0f : mn, f = __builtin_amdgcn_exp2f(mx - ref);
        mx = mn;
        L *= f;
        acc *= f;
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (j0 + i * SG >= np) break;   // (a repeated one may hold what is not finite)
            const float e = __builtin_amdgcn_exp2f(pm[i] - ref);
            L += pl[i] * e;
            acc += po[i] * e;
        }
    }
    if constexpr (SG > 1) {
        constexpr int LPR = DH / 4;
        __shared__ __attribute__((aligned(16))) f32x4 so[SG][LPR];
        __shared__ float sm[SG], sl[SG];
        so[sg][d4] = acc;
        if (d4 == 0) {
            sm[sg] = mx;
            sl[sg] = L;
        }
        __syncthreads();
        if (sg) return acc;
        float M = sm[0];
        for (int k = 1; k < SG; k++) M = fmaxf(M, sm[k]);
        const float ref = M == -INFINITY ? 0.0f : M;
        L = 0.0f;
        acc = f32x4{};
        for (int k = 0; k < SG; k++) {
            const float f = __builtin_amdgcn_exp2f(sm[k] - ref);
            L += sl[k] * f;
            acc += so[k][d4] * f;
        }
    }
    return np ? acc / L : f32x4{};
}

// ---- work split ------------------------------------------------------------------

constexpr int RW_WGS = 512;   // work-groups of a call to aim for: two per CU

inline int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

constexpr int RW_PLAN_TP = 32;   // (a plan serves both cache types)

// Microseconds of a call whose items, of up to `seen` positions, are one
// work-group of eight waves each (`wgs` of them): its start and end, its
// positions' steps and bytes (more than one per CU take turns).
inline double rows_together(double wgs, double seen, int d_head, int kv_f16)
{
    return 4.3 + 0.0019 * seen + 11e-6 * seen * d_head * (kv_f16 ? 4 : 8) * std::max(1.0, wgs / 256);
}
// CMOL_SESSION_WHOLE=0 / 1: items in pieces / whole wherever there is a choice
// (-1: by what both are estimated to cost).
int rows_whole_env();
// Pieces for n items of up to `span` tiles on `heads` work-groups each, to make
// `wgs` work-groups; 0 where the items alone fill the chip.
int rows_plan_bal(int n, long heads, long span, long wgs);

// What a call of these shapes splits into, and the number of its partial
// results.
struct RowsPlan {
    int bal = 0, parts = 0;
    size_t pieces = 0, cross = 0;   // pm / pl / po, and xm / xl / xo
    size_t split = 0;               // bytes of the f16 pairs
};
RowsPlan rows_plan_window(int n, int n_heads, int n_kv, int d_head, int max_ctx, int window, int sinks);
RowsPlan rows_plan_prompt(int n, int n_heads, int n_kv, int d_head, int max_ctx, int window, int sinks);
RowsPlan rows_plan_shared(int n, int n_heads, int n_kv, int d_head, int prefix, int max_ctx);

int launch_attn_window(const RowsArgs &a, hipStream_t s);   // (with a.prefix: behind it, every item whole)
int launch_attn_window_prompt(const RowsArgs &a, hipStream_t s);
int launch_attn_shared(const RowsArgs &a, hipStream_t s);

// Prompts whose query rows share the positions through LDS (attn_wprompt.hip),
// WP_ROWS per work-group; d_head 64 and 128.
constexpr int WP_ROWS = 128;
bool wprompt_takes(int d_head);
size_t wprompt_split_bytes(int n, int n_kv, int d_head, int max_ctx, int window, int sinks);
int launch_wprompt(const RowsArgs &a, hipStream_t s);

#define RW_BY_D_HEAD(d, F)          \
    switch (d) {                    \
    case 16: F(16) break;           \
    case 32: F(32) break;           \
    case 64: F(64) break;           \
    case 128: F(128) break;         \
    case 256: F(256) break;         \
    default: return -4;             \
    }
