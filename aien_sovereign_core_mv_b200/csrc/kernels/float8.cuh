// A block's scale and codes, for every kernel that leaves numbers in 8 bits (float8_rows.cu says what they are).
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace aien {

constexpr int F8_BLOCK = 128;
constexpr float F8_TOP = 448.0f, F8_LEAST = 1.17549435e-38f;      // the largest e4m3 number; 2^-126

__device__ __forceinline__ uint32_t f8_bits(float v) { return __float_as_uint(fabsf(v)); }
__device__ __forceinline__ float f8_scale(uint32_t top) {
    return top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fmaxf(__uint_as_float(top) * (1.0f / F8_TOP), F8_LEAST);
}
// One instruction of the special-function unit, at most a unit off; a scale and its reciprocal are ordinary numbers (2^-126 to 2^120).
__device__ __forceinline__ float f8_reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float f8_inverse(float scale) { return f8_reciprocal(scale); }
// act(g) * u: silu, or the gelu in its tanh form, from one exponential and one reciprocal (for large -g the exponential is infinite, its reciprocal 0).
template <bool GELU>
__device__ __forceinline__ float f8_gate(float g, float u) {
    if (GELU) return 0.5f * g * (1.0f + tanh_ex2(0.7978845608028654f * (g + 0.044715f * g * g * g))) * u;
    float t;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(g * -1.4426950408889634f));
    return g * f8_reciprocal(1.0f + t) * u;
}
__device__ __forceinline__ uint32_t f8_pair(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 f8_pack(const float v[8], float inv) {
    return make_uint2(f8_pair(v[0] * inv, v[1] * inv) | f8_pair(v[2] * inv, v[3] * inv) << 16,
                      f8_pair(v[4] * inv, v[5] * inv) | f8_pair(v[6] * inv, v[7] * inv) << 16);
}

}  // namespace aien
