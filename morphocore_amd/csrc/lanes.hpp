// Sums over neighbouring lanes on the vector unit (norm.hip, rotary.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mca
{

// A sum (float or double) as the 32-bit registers that lane exchanges move.
template <typename S>
struct Words
{
    static constexpr int N = sizeof(S) / 4;
    uint32_t w[N];
};

template <int CTRL, typename S>
__device__ __forceinline__ S dpp_add(S s)
{
    Words<S> a = __builtin_bit_cast(Words<S>, s);
#pragma unroll
    for (int i = 0; i < a.N; ++i) a.w[i] = (uint32_t)__builtin_amdgcn_mov_dpp((int)a.w[i], CTRL, 0xf, 0xf, true);
    return s + __builtin_bit_cast(S, a);
}

template <bool HALVES, typename S>
__device__ __forceinline__ S swap_add(S s)
{
    Words<S> a = __builtin_bit_cast(Words<S>, s), b = a;
#pragma unroll
    for (int i = 0; i < a.N; ++i)
    {
        const auto t = HALVES ? __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false) : __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
        a.w[i] = t[0], b.w[i] = t[1];
    }
    return __builtin_bit_cast(S, a) + __builtin_bit_cast(S, b);
}

// The sum over G consecutive lanes (a power of two up to the wave), in every one of them, on the vector unit.
template <int G, typename S>
__device__ __forceinline__ S lane_sum(S s)
{
    if constexpr (G > 1) s = dpp_add<0xb1>(s);   // lane ^ 1
    if constexpr (G > 2) s = dpp_add<0x4e>(s);   // lane ^ 2
    if constexpr (G > 4) s = dpp_add<0x141>(s);  // the other 4 of 8 (mirrored)
    if constexpr (G > 8) s = dpp_add<0x140>(s);  // the other 8 of 16 (mirrored)
    if constexpr (G > 16) s = swap_add<false>(s);
    if constexpr (G > 32) s = swap_add<true>(s);
    return s;
}

}  // namespace mca
