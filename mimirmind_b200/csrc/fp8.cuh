// Layer weights in 8 bits: what the quantisation and the products over blocks of 128 share.
//
// A row is held as e4m3 numbers q with one fp32 scale s per block of 128 (the last block may be shorter), x ~ q s:
//   s = max(fl(largest |x| / 448), 2^-126),   q = e4m3(fl(x / s)) (to nearest, ties to even; |x / s| never rounds above 448).
// 2^-126 keeps s a normal number for blocks of noughts and of numbers near the type's smallest.  A NaN in a block makes s and every
// q of it NaN; an infinity makes s infinite and its own q NaN: both reach the whole row of a product, and no other row.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

constexpr int FP8_BLOCK = 128;

// |v| as bits: they order as the numbers do, with NaN above infinity, so that a maximum keeps a NaN
__device__ __forceinline__ uint32_t fp8_size_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float fp8_scale_of(uint32_t largest_bits) {
    const float s = __fdiv_rn(__uint_as_float(largest_bits), 448.0f);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;      // a NaN stays
}

__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
__device__ __forceinline__ uint8_t fp8_one(float a) { return (uint8_t)__nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E4M3); }

__device__ __forceinline__ float fp8_to_f32(uint8_t v) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)v, __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
}

// glu_act, with a NaN in either half kept (the clamped form's minimum and maximum would lose it)
__device__ __forceinline__ float fp8_glu(float g, float u, int act, float limit, float s) {
    const float h = glu_act<false>(g, u, act, limit, s);
    return g != g || u != u ? __uint_as_float(0x7fffffffu) : h;
}
