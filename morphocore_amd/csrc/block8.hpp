// Rows of values in units and 8-bit blocks, shared by the channel-mixing kernels (norm.hip, gated.hip,
// weight8.hip).
//
// A lane holds a unit of 8 consecutive values of a row in float32; 4 consecutive lanes hold a block of 32.
// A block is kept in 8 bits as 32 codes and one scale byte b: value = e4m3(code) * 2^(b - 127). The
// exponent is the smallest with max |v| <= 448 * 2^(b - 127) (448: the largest e4m3 value) over the block's
// finite values, so nothing saturates, within [-117, 119]: from 2^-117 on every code's value is a normal
// float32 and bfloat16 (the smallest code is 2^-9), and above 448 * 2^119 values saturate, since a larger
// scale would round the largest float32 values up to infinity. NaN and infinities become the NaN code.
// e4m3 has 4 significant bits, so a value is exact in bfloat16; the code layout and the scale byte are
// those of the OCP microscaling formats (E4M3 elements, E8M0 scales, blocks of 32), which gfx950 converts
// in one instruction for two values (v_cvt_scalef32_*).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.hpp"

namespace mca
{

constexpr int UNIT = 8;
constexpr int MX_BLOCK = 32;
constexpr int MX_LANES = MX_BLOCK / UNIT;
constexpr int SCALE_MIN = 127 - 117, SCALE_MAX = 127 + 119;
constexpr uint32_t LARGEST_BITS = 0x7f600000;  // 448 * 2^119
constexpr float LARGEST = 0x1.cp127f;

inline __host__ __device__ int units_of(int cols) { return (int)(((int64_t)cols + UNIT - 1) / UNIT); }
inline __host__ __device__ int blocks_of(int cols) { return (int)(((int64_t)cols + MX_BLOCK - 1) / MX_BLOCK); }

// Whether a launch that moves `bytes` writes past the caches: where they are more than the last-level cache (256 MB)
// holds, the results are gone from it before they are read, and streaming stores leave what they would
// displace (8192 x 4096 bfloat16 norm with residual: 46 us, 56 without). Below, a reader finds them there.
inline bool streams(double bytes) { return bytes > 256e6; }

// A unit as stored: 8 values in consecutive dwords (two 16-bit values each), which keeps a unit that waits in
// registers as small as it is in memory.
template <typename T>
struct RawUnit
{
    static constexpr int DWORDS = UNIT * (int)sizeof(T) / 4;
    uint32_t d[DWORDS];

    __device__ __forceinline__ float operator[](int j) const
    {
        if constexpr (sizeof(T) == 4)
            return __uint_as_float(d[j]);
        else if constexpr (std::is_same_v<T, __bf16>)
            return __uint_as_float(j % 2 ? d[j / 2] & 0xffff0000u : d[j / 2] << 16);
        else
            return (float)__builtin_bit_cast(_Float16, (uint16_t)(d[j / 2] >> (16 * (j % 2))));
    }

    // Rounded to nearest even.
    __device__ __forceinline__ void set(const float (&v)[UNIT])
    {
#pragma unroll
        for (int i = 0; i < DWORDS; ++i)
        {
            if constexpr (sizeof(T) == 4)
            {
                d[i] = __float_as_uint(v[i]);
            }
            else
            {
                typedef float f2 __attribute__((ext_vector_type(2)));
                typedef T t2 __attribute__((ext_vector_type(2)));
                const f2 pair = {v[2 * i], v[2 * i + 1]};
                d[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, t2));
            }
        }
    }

    // n values down, zeros above.
    __device__ __forceinline__ void shift(int n)
    {
        constexpr int PER = 4 / (int)sizeof(T);  // values of a dword
#pragma unroll
        for (int s = 4; s >= PER; s /= 2)
            if (n & s)
            {
#pragma unroll
                for (int i = 0; i < DWORDS; ++i) d[i] = i + s / PER < DWORDS ? d[i + s / PER] : 0;
            }
        if constexpr (PER == 2)
            if (n & 1)
            {
#pragma unroll
                for (int i = 0; i < DWORDS; ++i) d[i] = d[i] >> 16 | (i + 1 < DWORDS ? d[i + 1] << 16 : 0);
            }
    }
};

// The 8 values from column c of a row on, p the first of them, `valid` = the columns from c to the row's end:
// those beyond it are 0. p is aligned to T only: global accesses of gfx950 take any alignment, so rows of
// odd widths load as wide as others. A row's last, partial unit is read as the row's last 8 values, which
// are then moved down (a row of fewer than 8 is read value by value).
template <typename T>
__device__ __forceinline__ void load_raw(const T* __restrict__ p, int c, int valid, RawUnit<T>& raw)
{
    if (valid >= UNIT)
    {
        __builtin_memcpy(raw.d, p, sizeof(raw.d));
        return;
    }
#pragma unroll
    for (int i = 0; i < RawUnit<T>::DWORDS; ++i) raw.d[i] = 0;
    if (valid <= 0) return;
    if (c > 0)
    {
        __builtin_memcpy(raw.d, p - (UNIT - valid), sizeof(raw.d));
        raw.shift(UNIT - valid);
        return;
    }
#pragma unroll
    for (int j = 0; j < UNIT - 1; ++j)
        if (j < valid)
        {
            if constexpr (sizeof(T) == 4)
                raw.d[j] = __builtin_bit_cast(uint32_t, p[j]);
            else
                raw.d[j / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[j]) << (16 * (j % 2));
        }
}

template <typename T>
__device__ __forceinline__ void load_unit(const T* __restrict__ p, int c, int valid, float (&v)[UNIT])
{
    RawUnit<T> raw;
    load_raw(p, c, valid, raw);
#pragma unroll
    for (int j = 0; j < UNIT; ++j) v[j] = raw[j];
}

// streaming: past the caches (see streams()).
template <typename T>
__device__ __forceinline__ void store_unit(T* __restrict__ p, int valid, const float (&v)[UNIT], bool streaming = false)
{
    RawUnit<T> raw;
    raw.set(v);
    if (valid >= UNIT)
    {
        if (streaming)
        {
            typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
            typedef u32x4 unaligned_u32x4 __attribute__((aligned(2)));
#pragma unroll
            for (int i = 0; i < RawUnit<T>::DWORDS; i += 4)
            {
                const u32x4 q = {raw.d[i], raw.d[i + 1], raw.d[i + 2], raw.d[i + 3]};
                __builtin_nontemporal_store(q, (unaligned_u32x4*)((uint32_t*)p + i));
            }
        }
        else
        {
            __builtin_memcpy(p, raw.d, sizeof(raw.d));
        }
        return;
    }
    // The rest of a row in pieces of 4, 2 and 1 values.
    if (valid <= 0) return;
    if (valid & 4)
    {
        __builtin_memcpy(p, raw.d, 4 * sizeof(T));
        raw.shift(4);
    }
    if (valid & 2)
    {
        __builtin_memcpy(p + (valid & 4), raw.d, 2 * sizeof(T));
        raw.shift(2);
    }
    if (valid & 1) __builtin_memcpy(p + (valid & 6), raw.d, sizeof(T));
}

// v rounded to T and back: what a reader of the stored value sees.
template <typename T>
__device__ __forceinline__ void round_unit(float (&v)[UNIT])
{
    RawUnit<T> raw;
    raw.set(v);
#pragma unroll
    for (int j = 0; j < UNIT; ++j) v[j] = raw[j];
}

// The same of codes.
__device__ __forceinline__ uint2 load_codes(const uint8_t* __restrict__ p, int c, int valid)
{
    uint64_t q = 0;
    if (valid >= UNIT)
    {
        __builtin_memcpy(&q, p, sizeof(q));
    }
    else if (valid > 0 && c > 0)
    {
        __builtin_memcpy(&q, p - (UNIT - valid), sizeof(q));
        q >>= 8 * (UNIT - valid);
    }
    else
    {
#pragma unroll
        for (int j = 0; j < UNIT - 1; ++j)
            if (j < valid) q |= (uint64_t)p[j] << (8 * j);
    }
    return make_uint2((uint32_t)q, (uint32_t)(q >> 32));
}

__device__ __forceinline__ void store_codes(uint8_t* __restrict__ p, int valid, uint2 c)
{
    if (valid >= UNIT)
    {
        __builtin_memcpy(p, &c, sizeof(c));
        return;
    }
    uint32_t w = c.x;
    if (valid & 4)
    {
        __builtin_memcpy(p, &w, 4);
        w = c.y;
    }
    if (valid & 2)
    {
        __builtin_memcpy(p + (valid & 4), &w, 2);
        w >>= 16;
    }
    if (valid & 1) p[valid & 6] = (uint8_t)w;
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// The largest magnitude's bits over the block; every lane of the block calls it.
__device__ __forceinline__ uint32_t block_largest(const float (&v)[UNIT])
{
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < UNIT; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));         // lane ^ 1
    return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));      // lane ^ 2
}

typedef short short2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float scale)
{
    short2v r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
    return __builtin_bit_cast(uint32_t, r);
}

// The unit's codes, and the block's scale byte. Values beyond a row's end are passed as 0.
__device__ __forceinline__ uint2 pack_unit(const float (&in)[UNIT], uint32_t& byte)
{
    float v[UNIT];
#pragma unroll
    for (int j = 0; j < UNIT; ++j) v[j] = in[j];
    uint32_t m = block_largest(v);
    if (m > LARGEST_BITS)  // saturating, infinite or NaN values: the whole block's lanes come here
    {
        float f[UNIT];
#pragma unroll
        for (int j = 0; j < UNIT; ++j)
        {
            const bool finite = (__float_as_uint(v[j]) & 0x7fffffffu) < 0x7f800000u;
            f[j] = finite ? fminf(fmaxf(v[j], -LARGEST), LARGEST) : 0.0f;
            v[j] = finite ? f[j] : __builtin_nanf("");
        }
        m = block_largest(f);
    }
    // 448 = 1.75 * 2^8: the biased exponent less 8, one more for significands above 1.75.
    byte = (uint32_t)clampi((int)((m + 0x1fffffu) >> 23) - 8, SCALE_MIN, SCALE_MAX);
    const float scale = scale_of(byte);
    return make_uint2(pack4(v[0], v[1], v[2], v[3], scale), pack4(v[4], v[5], v[6], v[7], scale));
}

__device__ __forceinline__ void unpack_unit(uint2 c, float scale, float (&v)[UNIT])
{
    const float2v a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, scale, true);
    const float2v d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, scale, false), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, scale, true);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = d.x, v[5] = d.y, v[6] = e.x, v[7] = e.y;
}

// Codes and scales of one unit written to a packed row (codes, scales: the row's first).
__device__ __forceinline__ void store_packed(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int unit, int valid,
                                             const float (&v)[UNIT])
{
    uint32_t byte;
    const uint2 c = pack_unit(v, byte);
    if (valid > 0)
    {
        store_codes(codes + (int64_t)unit * UNIT, valid, c);
        if (unit % MX_LANES == 0) scales[unit / MX_LANES] = (uint8_t)byte;
    }
}

}  // namespace mca
