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
constexpr int FP8_MAX = 1 << 30;      // rows, columns and depths stay below: places behind their ends are still ints

// |v| as bits: they order as the numbers do, with NaN above infinity, so that a maximum keeps a NaN
__device__ __forceinline__ uint32_t fp8_size_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float fp8_scale_of(uint32_t largest_bits) {
    const float s = __fdiv_rn(__uint_as_float(largest_bits), 448.0f);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;      // a NaN stays
}

// v[i] = fl(v[i] / s).  The quotient by Markstein's division theorem (P. Markstein, Computation of elementary functions on the IBM RISC
// System/6000 processor, 1990): with r = fl(1 / s) and q = fl(v r), fl(q + r (v - q s)) is v / s rounded, as long as the remainder is no
// subnormal that lost bits: s of 2^-80 and more, where numbers so small that it is (below 2^-100) come out as nought in e4m3 either way.
// Smaller and very large scales are brought there first, with their numbers, by a power of two: what a large one's numbers lose that way (below 2^-62 of them)
// is nought in e4m3 too.  An infinite s gives nought for a finite number and NaN for an infinite one, as the division does.
template <int N>
__device__ __forceinline__ void fp8_quotients(float* v, float s) {
    if (!(s >= 8.27180613e-25f && s < 1e30f)) {
        const float k = s < 1.0f ? 18446744073709551616.0f : 5.42101086e-20f;      // 2^64, 2^-64
        s *= k;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= k;
    }
    const float r = __fdiv_rn(1.0f, s), d = r == 0.0f ? 0.0f : s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float q = v[i] * r;
        v[i] = fmaf(fmaf(-q, d, v[i]), r, q);
    }
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

// eight numbers from a 16-byte boundary
template <typename T>
__device__ __forceinline__ void fp8_load8(const T* p, float* v);
template <>
__device__ __forceinline__ void fp8_load8<float>(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <>
__device__ __forceinline__ void fp8_load8<__nv_bfloat16>(const __nv_bfloat16* p, float* v) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// The gated activations of glu_act for values that are quantised or rounded to 16 bits next: exponentials and quotients of about 2^-20
// instead of 2^-23.  A NaN in either half is
// kept, also where the clamped form's minimum and maximum would lose it.
template <int ACT>
__device__ __forceinline__ float fp8_glu_as(float g, float u, float limit, float s) {
    g *= s;
    u *= s;
    if (ACT == MM_GLU_CLAMPED) {
        const float top = fminf(g, limit), v = fminf(fmaxf(u, -limit), limit) + 1.0f;
        const float h = __fdividef(top, 1.0f + __expf(-MM_GLU_CLAMPED_ALPHA * top)) * v;
        return g != g || u != u ? __uint_as_float(0x7fffffffu) : h;
    }
    // gelu(g) = g / (1 + exp(-2 c (g + 0.044715 g^3))), c = sqrt(2 / pi)
    const float z = ACT == MM_GLU_GELU_TANH ? 1.5957691216057308f * (g + 0.044715f * g * g * g) : g;
    return __fdividef(g, 1.0f + __expf(-z)) * u;
}
__device__ __forceinline__ float fp8_glu(float g, float u, int act, float limit, float s) {
    return act == MM_GLU_SILU ? fp8_glu_as<MM_GLU_SILU>(g, u, limit, s)
                              : act == MM_GLU_CLAMPED ? fp8_glu_as<MM_GLU_CLAMPED>(g, u, limit, s) : fp8_glu_as<MM_GLU_GELU_TANH>(g, u, limit, s);
}
