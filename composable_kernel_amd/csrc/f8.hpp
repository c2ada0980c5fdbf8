// 8-bit operands: conversions between e4m3 / int8 codes and 16- or 32-bit floats, shared by the serving kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "gemm_tile.hpp"

namespace ckx {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kE4m3Max  = 448.0f;
constexpr float kI8Max    = 127.0f;
constexpr float kTinyAmax = 7.888609052210118e-31f; // 2^-100: the least magnitude a scale is made for, so that 1 / scale is finite
constexpr int kGroup      = 128;                    // columns that share a scale

enum CodeType
{
    CODE_E4M3 = 0,
    CODE_I8   = 1
};

// two codes (bytes 2 * HI, 2 * HI + 1 of w) as a pair of T: exact for either code (e4m3 has 4 significant bits, int8 at most
// 8, bf16 holds 8 and fp16 11; the ranges fit)
template <int CODE, typename T, bool HI>
__device__ __forceinline__ uint32_t code_pair(uint32_t w)
{
    if constexpr(CODE == CODE_E4M3)
    {
        if constexpr(std::is_same<T, __bf16>::value)
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, HI));
        else
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
    }
    else
    {
        const float lo = (float)(int8_t)(w >> (HI ? 16 : 0)), hi = (float)(int8_t)(w >> (HI ? 24 : 8));
        if constexpr(std::is_same<T, __bf16>::value) // (exact: the upper halves)
            return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
        else
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
    }
}
// eight codes -> eight T
template <int CODE, typename T>
__device__ __forceinline__ i32x4 codes8(uint32_t lo, uint32_t hi)
{
    return i32x4{(int)code_pair<CODE, T, false>(lo), (int)code_pair<CODE, T, true>(lo), (int)code_pair<CODE, T, false>(hi),
                 (int)code_pair<CODE, T, true>(hi)};
}
// one code as a float
template <int CODE>
__device__ __forceinline__ float code_value(uint32_t w, int byte)
{
    if constexpr(CODE == CODE_I8)
        return (float)(int8_t)(w >> (8 * byte));
    else
    {
        switch(byte)
        {
        case 0: return __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
        case 1: return __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
        case 2: return __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
        default: return __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
        }
    }
}
// four floats -> four codes, round to nearest even. The values lie within the code's range (up to a rounding of its end).
template <int CODE>
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d)
{
    if constexpr(CODE == CODE_E4M3)
    {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    }
    else
        return (uint32_t)pack4_low_bytes((int)__builtin_rintf(a), (int)__builtin_rintf(b), (int)__builtin_rintf(c),
                                         (int)__builtin_rintf(d));
}

// x * f / d, the quotient rounded once: a multiplication by 1 / d leaves it up to two roundings off, which turns codes over where it
// lies half way between two of them, and with x of 16 bits that is no rarity (x = 0.75 of the group's largest is such a place). The
// remainder of the first quotient is exact, so that the second is the nearest. f is a few bits long: x * f is exact for 16-bit types,
// its rest is added for fp32 (EXACT false). d infinite: 0 (NaN for an infinite x); d NaN: NaN.
struct Quotient
{
    float f, d, inv;
    __device__ __forceinline__ Quotient(float f_, float d_) : f(f_), d(__builtin_isinf(d_) ? 0.0f : d_), inv(1.0f / d_) {}
    template <bool EXACT>
    __device__ __forceinline__ float of(float x) const
    {
        const float y = x * f, q = y * inv;
        float rest = __builtin_fmaf(-q, d, y);
        if constexpr(!EXACT)
            rest += __builtin_fmaf(x, f, -y);
        return __builtin_fmaf(rest, inv, q);
    }
};
// x * Q / amax with Q the largest code: both brought down by a power of two, so that nothing overflows
template <int CODE>
__device__ __forceinline__ Quotient quotient_of(float amax)
{
    return CODE == CODE_E4M3 ? Quotient(kE4m3Max / 512, amax * (1.0f / 512)) : Quotient(kI8Max / 128, amax * (1.0f / 128));
}

// eight consecutive elements of T as floats, at any address
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8])
{
    if constexpr(sizeof(T) == 4)
    {
        const f32x4 a = load_vec<f32x4>(p), b = load_vec<f32x4>(p + 4);
#pragma unroll
        for(int i = 0; i < 4; ++i)
            x[i] = a[i], x[4 + i] = b[i];
    }
    else
    {
        typedef T tx8 __attribute__((ext_vector_type(8)));
        const tx8 a = load_vec<tx8>(p);
#pragma unroll
        for(int i = 0; i < 8; ++i)
            x[i] = (float)a[i];
    }
}

} // namespace ckx
