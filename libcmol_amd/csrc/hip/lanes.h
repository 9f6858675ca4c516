// lanes.h — reductions over the lanes of a wave by DPP and lane swaps.  A
// ds_bpermute, which __shfl_xor is, takes about 130 cycles there and back; a step
// here is two or three vector instructions, and a reduction over 64 lanes is a
// long chain in kernels that run a few microseconds (5 sessions behind a prefix
// of 777: 9.55 us with shuffles, 8.7; logits of 8 rows 7.75, 7.2; of 32 rows with
// all penalties 17.5, 16.9).
#pragma once
#include "common.h"

template <int CTRL>
__device__ __forceinline__ uint32_t lane_dpp(uint32_t x)
{
    return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float lane_dpp(float x)
{
    return __uint_as_float(lane_dpp<CTRL>(__float_as_uint(x)));
}

// The value of the lane O away (lane ^ O), O below 16.  (To be called by every
// lane: not inside a selection.)
template <int O, typename T>
__device__ __forceinline__ T lane_xor(T x)
{
    static_assert(O == 1 || O == 2 || O == 4 || O == 8, "within a row of 16");
    if constexpr (O == 1) return lane_dpp<0xb1>(x);                     // quad_perm 1 0 3 2
    else if constexpr (O == 2) return lane_dpp<0x4e>(x);                // quad_perm 2 3 0 1
    else if constexpr (O == 4) return lane_dpp<0x1b>(lane_dpp<0x141>(x));   // halves of a row mirrored, then quads
    else return lane_dpp<0x128>(x);                                     // row_ror 8
}

// f(x, the other's x) for the pairs of lanes O apart, f symmetric.
template <int O, typename F>
__device__ __forceinline__ uint32_t lanes_pair(uint32_t x, F f)
{
    if constexpr (O < 16) {
        return f(x, lane_xor<O>(x));
    } else {
        const auto y = O == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false)
                               : __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return f(y[0], y[1]);
    }
}
template <int O>
__device__ __forceinline__ float lanes_add(float x)
{
    return __uint_as_float(lanes_pair<O>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
template <int O>
__device__ __forceinline__ float lanes_max(float x)
{
    return __uint_as_float(lanes_pair<O>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}

// Inclusive sums over the lanes, and the whole wave's (uniform).
__device__ __forceinline__ unsigned wave_scan_u(unsigned v)
{
    v += lane_dpp<0x111>(v);   // row_shr 1, 2, 4, 8
    v += lane_dpp<0x112>(v);
    v += lane_dpp<0x114>(v);
    v += lane_dpp<0x118>(v);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast 31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ unsigned wave_sum_u(unsigned v)
{
    return __builtin_amdgcn_readlane(wave_scan_u(v), 63);
}
