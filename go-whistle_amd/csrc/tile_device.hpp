// Device helpers of the attention kernels whose tiles of keys and values pass
// through LDS to the 32x32 matrix instructions (cross_kernels.hip,
// rows_kernels.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cqhip {

using f32x16 = float __attribute__((ext_vector_type(16)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using s16x8 = short __attribute__((ext_vector_type(8)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using lds_bytes = __attribute__((address_space(3))) unsigned char;

template <int TYPE>
constexpr float kLift = TYPE == 1 ? 7.0f : 0.0f;  // log2 of the largest weight, before the lag of the maximum

template <int TYPE>
__device__ __forceinline__ f32x16 mfma16(s16x8 a, s16x8 b, f32x16 c) {
    if constexpr (TYPE == 1)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int TYPE>
__device__ __forceinline__ short round16(float x) {
    if constexpr (TYPE == 1)
        return __builtin_bit_cast(short, static_cast<_Float16>(x));
    else
        return __builtin_bit_cast(short, static_cast<__bf16>(x));
}

// The first and the second parts of two weights.
template <int TYPE>
__device__ __forceinline__ uint32_t first_parts(float x, float y) {
    if constexpr (TYPE == 1)
        return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(x), static_cast<_Float16>(y)});
    else  // the upper halves
        return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);
}
template <int TYPE>
__device__ __forceinline__ uint32_t second_parts(float x, float y, uint32_t parts) {
    if constexpr (TYPE == 1) {  // x - part by a dot with (-1, 0): one instruction
        const f16x2 p = __builtin_bit_cast(f16x2, parts);
        const f16x2 lower = {static_cast<_Float16>(-1.0f), static_cast<_Float16>(0.0f)};
        const f16x2 upper = {static_cast<_Float16>(0.0f), static_cast<_Float16>(-1.0f)};
        return first_parts<1>(__builtin_amdgcn_fdot2(p, lower, x, false), __builtin_amdgcn_fdot2(p, upper, y, false));
    } else {
        const bf16x2 p = {static_cast<__bf16>(x - __uint_as_float(__float_as_uint(x) & 0xffff0000u)),
                          static_cast<__bf16>(y - __uint_as_float(__float_as_uint(y) & 0xffff0000u))};
        return __builtin_bit_cast(uint32_t, p);
    }
}

// Four pairs of 16-bit values, with 0 in place of infinities and NaNs.
template <int TYPE>
__device__ __forceinline__ s16x8 finite16(s16x8 x) {
    constexpr short kExponent = TYPE == 1 ? 0x7c00 : 0x7f80;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (x[e] & kExponent) == kExponent ? 0 : x[e];
    return x;
}

// The larger of the two halves' values, in both.
__device__ __forceinline__ float halves_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int D>
__device__ __forceinline__ int k_swizzle(int row) {
    return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
    return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
}

}  // namespace cqhip
