// attn_wprompt.hip — windowed attention of prompts (attn_rows.h) at d_head 64
// and 128, where there are enough query rows to share the cached positions
// through LDS.
//
// Rows of a kv head are (token, head of the group), token-major.  A work-group
// of four waves takes 128 of them and a part of the tiles of 32 positions that
// their tokens see between them; wave w owns rows 32 w .. +31 (two tiles of 16).
// The next tile is copied into LDS by direct-to-LDS loads while the present one
// is used.
//   fp16 cache: K pieces of 1 KiB in the operand's order (16 positions
//     x 32 dimensions, gathered by the loads' addresses), V rows as cached, their
//     32-byte units XOR-swizzled by the row for the transposing reads
//     (ds_read_b64_tr_b16) of the second product.
//   fp32 cache: k_prompt_split lays the positions the prompt sees out
//     once per call as f16 pairs (x = hi + lo), both operands in their order.
//     A tile is scaled by powers of two that put its largest |K| and |V| into
//     [2^9, 2^10), so hi and lo are normal f16 numbers whatever the cache's
//     range: 22 bits of a value, 2^-33 of the tile's largest below.  Where a
//     position's largest is below 2^-12 of the tile's, every position of the
//     tile is scaled by itself (`wide`): what a row does not see, or gives no
//     weight, leaves no trace in what it sees.  The score takes K's exponent
//     back; V's goes into the exponent of the weight, whose softmax reference
//     then follows what reaches the output, and the weights' sum takes it out.
// Products are exact (lo.lo, below 2^-22 of each, is left out over fp32), sums
// fp32; the query is split as the walk's of attn_rows.h, the weights too.
// Of the four pairs of halves a product over fp16 has two (the cache's is one
// number), over fp32 three.  Bound by the matrix pipe and by the softmax's vector
// instructions beside it: 4096 tokens of 16/4 heads of 128, window 2048, fp32 (155
// GFLOP in products): 158 us, 0.98 PFLOP/s, where a large library product reaches
// 1.15; 700 tokens behind 5000, fp16 (24 GFLOP), 40.4 us, a start and an end of
// about 8 among them.  Why 128 rows: a tile read from LDS serves two row tiles a
// wave; 256 would leave short prompts too few work-groups.
#include "attn_rows.h"
#include "lds_limit.h"

constexpr int WP_NT = 256, WP_TP = 32;   // threads, positions of a tile

// Tiles of TP positions that a prompt's tokens see: `ns` of sinks, then the
// run from lo (where the sinks reach into it, one run from 0).
struct PromptTiles {
    int s, lo, ns;
    __host__ __device__ PromptTiles(int pos0, int window, int sinks, int tp)
    {
        lo = pos0 + 1 > window ? pos0 + 1 - window : 0;
        s = sinks;
        if (sinks > lo) s = lo = 0;
        ns = (s + tp - 1) / tp;
    }
    __host__ __device__ int count(int last, int tp) const { return ns + (last + tp - lo) / tp; }
};

// A split tile: K hi and lo pieces, V hi and lo pieces, WP_TP positions.  Its
// exponents are K's, V's, whether it is wide and the least of V's; for a wide
// one, K's and V's of each position less the tile's.
constexpr int WP_HEAD = 4, WP_POS = 2 * WP_TP;   // ints of a tile: all heads first, then the positions'
constexpr int WP_LEXP = 20;                      // the weights' sum is held in units of 2^20
constexpr int WP_FAR = 90;                       // most that V's exponents may differ by
template <int DH>
constexpr int wp_tile_halves() { return WP_TP * DH * 4; }

// Bound by its bytes (4096 positions of 4 kv heads of 128: 17 MB read, 34 with the
// pairs written and their maxima: 13 us); a work-group per tile and kv head, the
// rows read twice, once whole for the largest of each, once in operand order.
template <int DH>
__global__ __launch_bounds__(256) void k_prompt_split(RowsArgs a, _Float16 *dst, int *exps, int tiles)
{
#pragma clang fp contract(off)
    constexpr int KS = DH / 32, DT = DH / 16, NK = 2 * KS * 64 / 256, NV = DT * 64 / 256, TH = wp_tile_halves<DH>();
    __shared__ float top[2][WP_TP];   // largest of each position's K, V
    const int tile = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x;
    const PromptTiles pt(a.pos0, a.window, a.sinks, WP_TP);
    const int p0 = tile < pt.ns ? tile * WP_TP : pt.lo + (tile - pt.ns) * WP_TP;
    const int cnt = min(WP_TP, (tile < pt.ns ? pt.s : a.pos0 + a.n) - p0);
    const size_t base = ((size_t)kvh * a.max_ctx + p0) * DH;
    const float *kb = (const float *)a.k + base, *vb = (const float *)a.v + base;
    dst += ((size_t)kvh * tiles + tile) * TH;
    float k[NK][8], v[NV][8];
#pragma unroll
    for (int j = 0; j < NK; j++) {
        const int it = tid + 256 * j, lane = it & 63, cs = it >> 6, c = cs / KS, s = cs % KS, p = 16 * c + (lane & 15);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const f32x4 x = p < cnt ? *(const f32x4 *)(kb + (size_t)p * DH + 32 * s + 8 * (lane >> 4) + 4 * h) : f32x4{};
#pragma unroll
            for (int e = 0; e < 4; e++) k[j][4 * h + e] = x[e];
        }
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int it = tid + 256 * j, lane = it & 63, t = it >> 6, g = lane >> 4;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int p = (e < 4 ? 0 : 12) + 4 * g + e;
            v[j][e] = p < cnt ? vb[(size_t)p * DH + 16 * t + (lane & 15)] : 0.0f;
        }
    }
    {   // eight threads per position
        const int p = tid >> 3;
        float tk = 0.0f, tv = 0.0f;
#pragma unroll
        for (int j = 0; j < DH / 32; j++) {
            const size_t at = (size_t)p * DH + 4 * ((tid & 7) + 8 * j);
            const f32x4 x = p < cnt ? *(const f32x4 *)(kb + at) : f32x4{}, y = p < cnt ? *(const f32x4 *)(vb + at) : f32x4{};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (fabsf(x[e]) < INFINITY) tk = fmaxf(tk, fabsf(x[e]));
                if (fabsf(y[e]) < INFINITY) tv = fmaxf(tv, fabsf(y[e]));
            }
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            tk = fmaxf(tk, __shfl_xor(tk, o, 64));
            tv = fmaxf(tv, __shfl_xor(tv, o, 64));
        }
        if ((tid & 7) == 0) {
            top[0][p] = tk;
            top[1][p] = tv;
        }
    }
    __syncthreads();
    // lanes 0 .. 31: K of a position, 32 .. 63: V (positions of zeros do not make a
    // tile wide; theirs is an exponent that raises no reference of ordinary values)
    auto exponent = [](float x) { return x > 0.0f ? max(ilogbf(x), -100) - 9 : -45; };
    const int own = tid & 63;
    const float mine = top[own >> 5][own & 31];
    float most = mine, least = mine > 0.0f ? mine : INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        most = fmaxf(most, __shfl_xor(most, o, 64));
        least = fminf(least, __shfl_xor(least, o, 64));
    }
    const bool wide = __ballot(least < most * 0x1p-12f) != 0;
    const int em = exponent(most), ex[2] = {__builtin_amdgcn_readlane(em, 0), __builtin_amdgcn_readlane(em, 32)};
    const size_t at = (size_t)kvh * tiles + tile;
    int low = wide && (own & 31) < cnt ? exponent(mine) : em;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor(low, o, 64));
    low = __builtin_amdgcn_readlane(low, 32);
    int *pos = exps + (size_t)a.n_kv * tiles * WP_HEAD + at * WP_POS;
    if (tid < WP_POS) {
        pos[tid] = wide ? exponent(mine) - em : 0;
        if (tid < WP_HEAD) exps[at * WP_HEAD + tid] = tid == 0 ? ex[0] : tid == 1 ? ex[1] : tid == 2 ? wide : low;
    }
    auto scale = [&](int i, int p) { return wide ? exponent(top[i][p]) : ex[i]; };
    auto put = [&](const float (&y)[8], _Float16 *to) {
        f16x8 hi, lo;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            hi[i] = (_Float16)y[i];
            lo[i] = (_Float16)(y[i] - (float)hi[i]);
        }
        *(f16x8 *)to = hi;
        *(f16x8 *)(to + 512) = lo;
    };
#pragma unroll
    for (int j = 0; j < NK; j++) {
        const int it = tid + 256 * j, e = scale(0, 16 * ((it >> 6) / KS) + (it & 15));
#pragma unroll
        for (int i = 0; i < 8; i++) k[j][i] = ldexpf(k[j][i], -e);
        put(k[j], dst + (it >> 6) * 1024 + (it & 63) * 8);
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int it = tid + 256 * j;
#pragma unroll
        for (int i = 0; i < 8; i++) v[j][i] = ldexpf(v[j][i], -scale(1, (i < 4 ? 0 : 12) + 4 * ((it & 63) >> 4) + i));
        put(v[j], dst + TH / 2 + (it >> 6) * 1024 + (it & 63) * 8);
    }
}

// LDS of a work-group: two stages of K and V.
template <int DH, bool F16>
constexpr int wp_lds() { return 2 * (F16 ? WP_TP * DH * 4 : wp_tile_halves<DH>() * 2); }

template <int DH, bool F16>
__global__ __launch_bounds__(WP_NT) __attribute__((amdgpu_waves_per_eu(2)))
void k_prompt_rows(RowsArgs a, const _Float16 *split, const int *exps, int tiles)
{
#pragma clang fp contract(off)
    typedef typename std::conditional<F16, _Float16, float>::type KT;
    constexpr int TP = WP_TP, CT = TP / 16, RT = 2;
    constexpr int KS = DH / 32, DT = DH / 16;
    constexpr int KB = F16 ? TP * DH * 2 : wp_tile_halves<DH>();   // K bytes of a tile (V: as many)
    constexpr int RPP = 1024 / (2 * DH);              // fp16: V rows per 1 KiB piece
    constexpr int VPW = TP / RPP / 4;                 // fp16: V pieces per wave
    extern __shared__ __attribute__((aligned(256))) uint8_t smem_w[];   // K [stage][KB], V the same
    __shared__ int odd, odd_row[WP_ROWS];

    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.n_heads / a.n_kv, rows = a.n * G;
    const int blocks = gridDim.x / a.n_kv;
    // the blocks of the longest lines first
    const int kvh = blockIdx.x % a.n_kv, r0 = (blocks - 1 - (int)(blockIdx.x / a.n_kv)) * WP_ROWS, part = blockIdx.y;
    const int nr = min(WP_ROWS, rows - r0);
    const int first = a.pos0 + r0 / G, last = a.pos0 + (r0 + nr - 1) / G;
    // the block's tiles: [0, na) and [nb, ne)
    const PromptTiles pt(a.pos0, a.window, a.sinks, TP);
    const int lo = max(first + 1 - a.window, 0);
    const int na = pt.s || !a.sinks ? pt.ns : (min(a.sinks, lo) + TP - 1) / TP;
    const int nb = max(pt.ns + (lo - pt.lo) / TP, na), ne = pt.count(last, TP);
    const int T = na + ne - nb, R = (T + a.parts - 1) / a.parts;
    const int u0 = min(part * R, T), u1 = min(u0 + R, T);
    auto tile = [&](int u) { return u < na ? u : u - na + nb; };
    auto start = [&](int t) { return t < pt.ns ? t * TP : pt.lo + (t - pt.ns) * TP; };
    auto limit = [&](int t) { return t < pt.ns ? pt.s : last + 1; };

    const size_t base = (size_t)kvh * a.max_ctx * DH;
    const uint8_t *kb = (const uint8_t *)uniform_ptr((const KT *)a.k + base);
    const uint8_t *vbp = (const uint8_t *)uniform_ptr((const KT *)a.v + base);
    const uint8_t *sb = (const uint8_t *)uniform_ptr(split + (size_t)kvh * tiles * wp_tile_halves<DH>());
    typedef const __attribute__((address_space(4))) int cint;   // (scalar loads)
    cint *ex = (cint *)uniform_ptr(exps + (size_t)kvh * tiles * WP_HEAD);
    const int *px = exps + (size_t)a.n_kv * tiles * WP_HEAD + (size_t)kvh * tiles * WP_POS;
    const int vrow = lane / (DH / 8), vch = lane % (DH / 8);
    uint8_t *const kl_ = smem_w, *const vl_ = smem_w + 2 * KB;
    auto issue_k = [&](int st, int u) {
        uint8_t *dst = kl_ + st * KB;
        const int t = tile(u);
        if constexpr (F16) {
            const int p0 = start(t), cnt = limit(t) - p0;   // (past it: its last position again)
            const uint8_t *ks = kb + (size_t)p0 * (2 * DH);
#pragma unroll
            for (int i = 0; i < CT * KS / 4; i++) {
                const int pc = wid * (CT * KS / 4) + i;   // 16 positions x 32 dimensions
                const uint32_t kp = (uint32_t)min(16 * (pc / KS) + col, cnt - 1) * (2 * DH) + 64 * (pc % KS) + 16 * g;
                __builtin_amdgcn_global_load_lds((const gvoid_t *)(ks + kp), (lvoid_t *)(dst + pc * 1024), 16, 0, 0);
            }
        } else {
            const uint8_t *src = sb + (size_t)t * (2 * KB);
#pragma unroll
            for (int i = 0; i < KB / 4096; i++) {
                const int pc = wid * (KB / 4096) + i;
                __builtin_amdgcn_global_load_lds((const gvoid_t *)(src + pc * 1024 + lane * 16), (lvoid_t *)(dst + pc * 1024),
                                                 16, 0, 0);
            }
        }
    };
    auto issue_v = [&](int st, int u) {
        uint8_t *dst = vl_ + st * KB;
        const int t = tile(u);
        if constexpr (F16) {
            const int p0 = start(t), cnt = limit(t) - p0;
            const uint8_t *vs = vbp + (size_t)p0 * (2 * DH);
#pragma unroll
            for (int i = 0; i < VPW; i++) {
                const int r = (wid * VPW + i) * RPP + vrow;   // row of the tile
                const int f = DH == 128 ? r & 7 : (r >> 1) & 3;
                const uint32_t vp = (uint32_t)min(r, cnt - 1) * (2 * DH) + 32 * ((vch >> 1) ^ f) + 16 * (vch & 1);
                __builtin_amdgcn_global_load_lds((const gvoid_t *)(vs + vp), (lvoid_t *)(dst + (wid * VPW + i) * 1024), 16, 0, 0);
            }
        } else {
            const uint8_t *src = sb + (size_t)t * (2 * KB) + KB;
#pragma unroll
            for (int i = 0; i < KB / 4096; i++) {
                const int pc = wid * (KB / 4096) + i;
                __builtin_amdgcn_global_load_lds((const gvoid_t *)(src + pc * 1024 + lane * 16), (lvoid_t *)(dst + pc * 1024),
                                                 16, 0, 0);
            }
        }
    };
    // K runs a tile ahead of V: the next tile's scores are computed beside the
    // present one's weights
    if (u0 < u1) {
        issue_k(0, u0);
        issue_v(0, u0);
    }

    auto row_at = [&](int r) {   // of q and out
        r = min(r0 + r, rows - 1);
        return (size_t)(r / G) * a.n_heads + (size_t)kvh * G + r % G;
    };
    // query operands of rows 32 wid + 16 rt + col: the row's largest into [2^9, 2^10)
    f16x8 qh[RT][KS], ql[RT][KS];
    float c2[RT];
    int pos[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int r = 32 * wid + 16 * rt + col;
        pos[rt] = a.pos0 + min(r0 + r, rows - 1) / G;
        const float *q = a.q + row_at(r) * DH + 8 * g;
        float x[KS][8], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const f32x4 y0 = ldg((const f32x4 *)(q + 32 * s)), y1 = ldg((const f32x4 *)(q + 32 * s + 4));
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[s][e] = e < 4 ? y0[e & 3] : y1[e & 3];
                top = fmaxf(top, fabsf(x[s][e]));
            }
        }
        top = lanes_max<32>(lanes_max<16>(top));
        const int e0 = top > 0.0f && top < INFINITY ? max(ilogbf(top), -100) - 9 : 0;
        c2[rt] = ldexpf(1.44269504088896341f / sqrtf((float)DH), e0);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = ldexpf(x[s][e], -e0);
                qh[rt][s][e] = (_Float16)y;
                ql[rt][s][e] = (_Float16)(y - (float)qh[rt][s][e]);
            }
    }
    // V of so many magnitudes in the block's tiles (whatever the part) that a
    // weight's sum could leave the range of fp32 beside another's contribution:
    // every row one by one
    bool far = false;
    int most = 0;
    if constexpr (!F16) {
        int least = 1000;
        most = -1000;
        for (int u = lane; u < T; u += 64) {
            most = max(most, ex[WP_HEAD * tile(u) + 1]);
            least = min(least, ex[WP_HEAD * tile(u) + 3]);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            most = max(most, __shfl_xor(most, o, 64));
            least = min(least, __shfl_xor(least, o, 64));
        }
        most = __builtin_amdgcn_readfirstlane(most);
        far = most > __builtin_amdgcn_readfirstlane(least) + WP_FAR;
        if (far) most = 0;
    }
    const f32x4 zero4 = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 o[RT][DT];
    float m[RT], mk[RT], l[RT];   // m: reference in log2 units (V's exponent with the score); mk = RW_SCALE - m
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m[rt] = -INFINITY;
        mk[rt] = RW_SCALE;
        l[rt] = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; t++) o[rt][t] = zero4;
    }
    // fp16: transposing reads, this lane's bytes of row 4g + col/4 (+ 16 per c)
    // of dimension tile t at vaddr ^ 32t
    const int vr = 4 * g + (col >> 2);
    const uint32_t vaddr = (uint32_t)(vr * (2 * DH) + 32 * (DH == 128 ? vr & 7 : (vr >> 1) & 3) + 8 * (col & 3));

    // operand pieces: q-th of a K tile (c = q / KS, s = q % KS), d-th of a V tile
    // (dimension tile d)
    static_assert(CT == 2, "two groups of 16 positions");
    constexpr int NP = F16 ? 1 : 2;
    auto read_k = [&](int st, int q, f16x8 (&x)[NP]) {
        const uint8_t *src = kl_ + st * KB + q * NP * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < NP; i++) x[i] = *(const f16x8 *)(src + i * 1024);
    };
    auto read_v = [&](int st, int d, f16x8 (&x)[NP]) {
        const uint8_t *src = vl_ + st * KB;
        if constexpr (F16) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4 ls16x4;
            src += vaddr ^ (32u * d);
            const s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls16x4 *)src);
            const s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls16x4 *)(src + 16 * (2 * DH)));
            x[0] = __builtin_bit_cast(f16x8, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
#pragma unroll
            for (int i = 0; i < NP; i++) x[i] = *(const f16x8 *)(src + (d * NP + i) * 1024 + lane * 16);
        }
    };
    // Products of two pieces with the row tiles' operands into y[piece][rt], those
    // with a low part first; consecutive ones on different sums.
    auto products = [&](const f16x8 (&x)[2][NP], const f16x8 *(&hi)[RT], const f16x8 *(&lo)[RT], f32x4 *(&y)[2][RT]) {
#pragma unroll
        for (int t = F16 ? 1 : 0; t < 3; t++)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
                    *y[i][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i][t == 0 ? NP - 1 : 0], t == 1 ? *lo[rt] : *hi[rt],
                                                                       *y[i][rt], 0, 0, 0);
    };
    auto score_step = [&](const f16x8 (&x)[2][NP], int s, f32x4 (&y)[RT][CT]) {   // k-step s of both c
        const f16x8 *hi[RT], *lo[RT];
        f32x4 *at[2][RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            hi[rt] = &qh[rt][s];
            lo[rt] = &ql[rt][s];
#pragma unroll
            for (int c = 0; c < CT; c++) {
                at[c][rt] = &y[rt][c];
                if (s == 0) y[rt][c] = zero4;
            }
        }
        products(x, hi, lo, at);
    };
    // sc[rt][c][i]: score of the tile's position 16c + 4g + i and row col
    f32x4 sc[RT][CT];
    __builtin_amdgcn_s_waitcnt(WAITCNT_VM_LGKM0(0));
    __syncthreads();
    if (u0 + 1 < u1) issue_k(1, u0 + 1);
    int ek = 0, ev = 0, wide = 0;   // of the tile
    if (u0 < u1) {
#pragma unroll
        for (int q = 0; q < KS; q++) {
            f16x8 k[2][NP];
            read_k(0, q, k[0]);
            read_k(0, KS + q, k[1]);
            score_step(k, q, sc);
        }
        if constexpr (!F16) {
            ek = ex[WP_HEAD * tile(u0)];
            ev = ex[WP_HEAD * tile(u0) + 1];
            wide = ex[WP_HEAD * tile(u0) + 2];
        }
    }
    for (int u = u0, st = 0; u < u1; u++, st ^= 1) {
        // K u + 1 and V u have landed, every wave is done with K u and V u - 1
        __builtin_amdgcn_s_waitcnt(WAITCNT_VM_LGKM0(0));
        __syncthreads();
        if (u + 2 < u1) issue_k(st, u + 2);
        if (u + 1 < u1) issue_v(st ^ 1, u + 1);
        const int t = tile(u), p0 = start(t), cnt = limit(t) - p0;
        float kf = 1.0f, ve = 0.0f, lk = 1.0f;
        int le = 0;   // lk = 2^le
        const int *alone = nullptr;   // (uniform) the positions' own exponents
        if constexpr (!F16) {
            kf = ldexpf(1.0f, ek);
            ve = (float)ev;
            le = -WP_LEXP - ev;
            lk = ldexpf(1.0f, le);
            if (wide) alone = px + (size_t)t * WP_POS + 4 * g;
            const int tn = tile(min(u + 1, u1 - 1));   // (its exponents in time)
            ek = ex[WP_HEAD * tn];
            ev = ex[WP_HEAD * tn + 1];
            wide = ex[WP_HEAD * tn + 2];
        }
        const int top = p0 + TP - 1;
        if (top > first || cnt < TP || (top >= a.sinks && p0 <= last - a.window)) {   // uniform
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int at = 16 * c + 4 * g + i, p = p0 + at;
                        if (at >= cnt || p > pos[rt] || (p >= a.sinks && p <= pos[rt] - a.window)) sc[rt][c][i] = -INFINITY;
                    }
        }
        // ---- online softmax: the reference
        float f[RT], mx[RT], mv[RT], ls[RT], lw[RT];
        bool up = false;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            // (above 0: a masked score times it stays -inf)
            f[rt] = F16 ? c2[rt] : fmaxf(c2[rt] * kf, 1e-37f);
            lw[rt] = 0.0f;
            if (!F16 && alone) {
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        sc[rt][c][i] = fmaf(ldexpf(sc[rt][c][i], alone[16 * c + i]), f[rt], (float)alone[WP_TP + 16 * c + i]);
                f[rt] = 1.0f;
            }
            mx[rt] = sc[rt][0][0];
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx[rt] = fmaxf(mx[rt], sc[rt][c][i]);
            mx[rt] = fmaf(mx[rt], f[rt], ve);
            up |= mx[rt] > m[rt] + RW_LAZY;
        }
        if (__ballot(up)) {   // (one branch for both row tiles: what follows is one block to schedule)
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                mx[rt] = lanes_max<32>(lanes_max<16>(mx[rt]));
                const float mn = fmaxf(m[rt], mx[rt]);
                const float mkn = mn == -INFINITY ? RW_SCALE : RW_SCALE - mn;
                const float al = m[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mkn - mk[rt]);
                m[rt] = mn;
                mk[rt] = mkn;
                l[rt] *= al;
#pragma unroll
                for (int d = 0; d < DT; d++) o[rt][d] *= al;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++) mv[rt] = mk[rt] + ve;
        if (!F16 && alone) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        lw[rt] += ldexpf(__builtin_amdgcn_exp2f(sc[rt][c][i] + mv[rt]), le - alone[WP_TP + 16 * c + i]);
            lk = 0.0f;
        }
        // ---- the weights (P, in two parts) between the next tile's scores, then
        // O^T += V^T P^T.  The order is fixed: a step's operand pieces are read
        // during the one before, and its products run beside its share of the weights'
        // instructions.  (A K stage past the last tile holds an old one: not used.)
        f32x4 sn[RT][CT];
        f16x8 kr[2][2][NP], ph[RT], pl[RT];
        constexpr int PAIRS = RT * CT * 2;
        auto weights = [&](int x) {   // scores 2x, 2x + 1 of (rt, c, i)
            const int rt = x / (CT * 2), c = x / 2 % CT, i = x % 2 * 2;
            const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[rt][c][i], f[rt], mv[rt]));
            const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[rt][c][i + 1], f[rt], mv[rt]));
            ls[rt] += e0 + e1;
            const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(e0, e1));
            const f16x2 lw = __builtin_bit_cast(
                f16x2, __builtin_amdgcn_cvt_pkrtz(fmaf((float)hi[0], -1.0f, e0), fmaf((float)hi[1], -1.0f, e1)));
            ph[rt][4 * c + i] = hi[0];
            ph[rt][4 * c + i + 1] = hi[1];
            pl[rt][4 * c + i] = lw[0];
            pl[rt][4 * c + i + 1] = lw[1];
        };
#pragma unroll
        for (int rt = 0; rt < RT; rt++) ls[rt] = 0.0f;
        // A wave with products ahead goes first: the other wave of its SIMD, at its
        // barrier, masks and reference, has the vector pipe while the matrix pipe is
        // fed (4096 tokens over fp32: 171 us without, 162 with the second product's
        // alone, 158; 700 over fp16: 41.7, 41.2, 40.4).
        __builtin_amdgcn_s_setprio(1);
        read_k(st ^ 1, 0, kr[0][0]);
        read_k(st ^ 1, KS, kr[0][1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < KS; q++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (q + 1 < KS) read_k(st ^ 1, i * KS + q + 1, kr[(q + 1) & 1][i]);
                else read_v(st, i, kr[(q + 1) & 1][i]);
            }
            score_step(kr[q & 1], q, sn);
#pragma unroll
            for (int x = q * PAIRS / KS; x < (q + 1) * PAIRS / KS; x++) weights(x);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++) l[rt] = F16 ? l[rt] + ls[rt] : fmaf(ls[rt], lk, l[rt]) + lw[rt];
#pragma unroll
        for (int d = 0; d < DT; d += 2) {
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (d + 2 < DT) read_v(st, d + 2 + i, kr[(KS + d / 2 + 1) & 1][i]);
            const f16x8 *hi[RT], *lo[RT];
            f32x4 *at[2][RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                hi[rt] = &ph[rt];
                lo[rt] = &pl[rt];
                at[0][rt] = &o[rt][d];
                at[1][rt] = &o[rt][d + 1];
            }
            products(kr[(KS + d / 2) & 1], hi, lo, at);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int c = 0; c < CT; c++) sc[rt][c] = sn[rt][c];
    }

    // ---- outputs: lane (col, g) holds dimensions 16d + 4g + i of row col
    if (tid == 0) odd = 0;
    if (tid < WP_ROWS) odd_row[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const float ls = lanes_add<32>(lanes_add<16>(l[rt]));
        const int r = 32 * wid + 16 * rt + col;
        const bool valid = r < nr;
        const float unit = F16 ? 1.0f : ldexpf(1.0f, -WP_LEXP), inv = unit / ls;
        const size_t at = ((size_t)kvh * rows + min(r0 + r, rows - 1)) * a.parts + part;
        f32x4 z = zero4;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const f32x4 y = o[rt][d] * (a.parts == 1 ? inv : unit);
            z += y * 0.0f;
            if (!valid) continue;
            if (a.parts == 1) *(f32x4 *)(a.out + row_at(r) * DH + 16 * d + 4 * g) = y;
            else *(f32x4 *)(a.xo + at * DH + 16 * d + 4 * g) = y;
        }
        if (valid && a.parts > 1 && g == 0) {
            a.xm[at] = m[rt] == -INFINITY ? -INFINITY : (F16 ? 0 : WP_LEXP) - mk[rt];   // of the weights as they are
            a.xl[at] = ls;
        }
        if (valid && (far || !(z[0] + z[1] + z[2] + z[3] + ls * 0.0f == 0.0f))) odd = odd_row[r] = 1;
    }
    // A masked position is in its tile's products with weight 0, which a V row
    // that is not finite turns into NaN for the rows that do not see it: rows
    // whose outputs are not finite are walked again one by one.
    __syncthreads();
    if (!odd) return;
    constexpr int DL = RowState<DH>::DL;
    for (int r = wid; r < nr; r += WP_NT / 64) {
        if (!odd_row[r]) continue;
        const size_t qa = row_at(r) * DH + lane * DL;
        const int p = a.pos0 + (r0 + r) / G;
        RowState<DH> s;
        s.m = -INFINITY;
        s.l = 0.0f;
#pragma unroll
        for (int d = 0; d < DL; d++) {
            s.q[d] = a.q[qa + d];
            s.o[d] = 0.0f;
        }
        for (int u = u0; u < u1; u++) {
            const int t = tile(u), p0 = start(t), end = min(min(p0 + TP, limit(t)), p + 1);
            row_walk<DH, KT>(s, (const KT *)a.k + base, (const KT *)a.v + base, p0, min(end, a.sinks));
            row_walk<DH, KT>(s, (const KT *)a.k + base, (const KT *)a.v + base,
                             max(max(p0, p + 1 - a.window), min(a.sinks, end)), end);
        }
        const size_t at = ((size_t)kvh * rows + r0 + r) * a.parts + part;
#pragma unroll
        for (int d = 0; d < DL; d++) {
            if (a.parts == 1) a.out[qa + d] = s.o[d] / s.l;
            else a.xo[at * DH + lane * DL + d] = ldexpf(s.o[d], -most);
        }
        if (a.parts > 1 && lane == 0) {   // (V's exponent in m, as in the parts that are not walked again)
            a.xm[at] = s.m + (float)most;
            a.xl[at] = ldexpf(s.l, -most);
        }
    }
}

bool wprompt_takes(int d_head) { return d_head == 64 || d_head == 128; }

// Bytes of the split copy: the tiles, and their exponents behind them.
size_t wprompt_split_bytes(int n, int n_kv, int d_head, int max_ctx, int window, int sinks)
{
    const long seen = std::min((long)max_ctx, (long)std::min(window, max_ctx) + std::min(sinks, max_ctx) + n);
    const size_t tiles = (size_t)n_kv * (ceil_div(seen, WP_TP) + 2);
    return tiles * (WP_TP * d_head * 8 + (WP_HEAD + WP_POS) * sizeof(int));
}

template <int DH, bool F16>
static int launch_dh(const RowsArgs &a, hipStream_t s)
{
    constexpr int LDS = wp_lds<DH, F16>();
    static LdsLimit limit;
    const bool ok = limit.raise(current_device(), [] {
        return hipFuncSetAttribute((const void *)k_prompt_rows<DH, F16>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) ==
               hipSuccess;
    });
    if (!ok) {
        (void)hipGetLastError();
        return -4;
    }
    int tiles = 0;
    _Float16 *split = (_Float16 *)a.split;
    int *exps = nullptr;
    if constexpr (!F16) {
        tiles = PromptTiles(a.pos0, a.window, a.sinks, WP_TP).count(a.pos0 + a.n - 1, WP_TP);
        exps = (int *)(split + (size_t)a.n_kv * tiles * wp_tile_halves<DH>());
        hipLaunchKernelGGL(k_prompt_split<DH>, dim3(tiles, a.n_kv), dim3(256), 0, s, a, split, exps, tiles);
    }
    const int blocks = ceil_div((long)a.n * (a.n_heads / a.n_kv), WP_ROWS);
    hipLaunchKernelGGL((k_prompt_rows<DH, F16>), dim3(a.n_kv * blocks, a.parts), dim3(WP_NT), LDS, s, a, split, exps, tiles);
    return 0;
}

int launch_wprompt(const RowsArgs &a, hipStream_t s)
{
    if (a.kv_f16) return a.d_head == 128 ? launch_dh<128, true>(a, s) : launch_dh<64, true>(a, s);
    return a.d_head == 128 ? launch_dh<128, false>(a, s) : launch_dh<64, false>(a, s);
}
