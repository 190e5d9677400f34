// Values of other lanes of a wave without LDS: DPP inside the rows of 16, gfx950's row swaps between them. A ds_bpermute takes
// some 100 cycles, these 8 to 16, which is what a chain of exchanges (a sort, a reduction) consists of.
#pragma once

#include "ql_device.h"

namespace ql {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}

typedef uint32_t u32pair __attribute__((ext_vector_type(2)));

// {v, v of lane ^ O} in either order, O = 16 or 32
template <int O>
__device__ __forceinline__ u32pair lane_pair(uint32_t v)
{
    static_assert(O == 16 || O == 32, "rows of 16 are swapped with their neighbours, or the halves");
    if constexpr (O == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return u32pair{r[0], r[1]};
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return u32pair{r[0], r[1]};
    }
}

// v of lane ^ O, for a power of two O below 64; lane: the wave's lane
template <int O>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane)
{
    if constexpr (O == 1) return dpp_u32<0xB1>(v);                       // quad_perm [1, 0, 3, 2]
    else if constexpr (O == 2) return dpp_u32<0x4E>(v);                  // quad_perm [2, 3, 0, 1]
    else if constexpr (O == 4) return dpp_u32<0x141>(dpp_u32<0x1B>(v));  // reversed in fours (^ 3), then in eights (^ 7)
    else if constexpr (O == 8) return dpp_u32<0x128>(v);                 // row_ror:8
    else {
        const u32pair p = lane_pair<O>(v);                               // first: v of the even row or lower half, in both
        return lane & O ? p.x : p.y;
    }
}

template <int O>
__device__ __forceinline__ float lane_xor_f(float v, int lane) { return __builtin_bit_cast(float, lane_xor<O>(__builtin_bit_cast(uint32_t, v), lane)); }
template <int O>
__device__ __forceinline__ uint64_t lane_xor64(uint64_t v, int lane)
{
    return (uint64_t)lane_xor<O>((uint32_t)(v >> 32), lane) << 32 | lane_xor<O>((uint32_t)v, lane);
}

// max and sum with the lane ^ 16 or ^ 32 (a bit cast of a vector's element itself gives the first one: copies)
template <int O>
__device__ __forceinline__ float pair_max(float v)
{
    const u32pair p = lane_pair<O>(__builtin_bit_cast(uint32_t, v));
    const uint32_t x = p.x, y = p.y;
    return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
template <int O>
__device__ __forceinline__ float pair_sum(float v)
{
    const u32pair p = lane_pair<O>(__builtin_bit_cast(uint32_t, v));
    const uint32_t x = p.x, y = p.y;
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
__device__ __forceinline__ float wave_max(float v, int lane)
{
    v = fmaxf(v, lane_xor_f<1>(v, lane));
    v = fmaxf(v, lane_xor_f<2>(v, lane));
    v = fmaxf(v, lane_xor_f<4>(v, lane));
    v = fmaxf(v, lane_xor_f<8>(v, lane));
    return pair_max<32>(pair_max<16>(v));
}
__device__ __forceinline__ float wave_sum(float v, int lane)
{
    v += lane_xor_f<1>(v, lane);
    v += lane_xor_f<2>(v, lane);
    v += lane_xor_f<4>(v, lane);
    v += lane_xor_f<8>(v, lane);
    return pair_sum<32>(pair_sum<16>(v));
}

}  // namespace ql
