// A block's scale and codes, for every kernel that leaves numbers in 8 bits (float8_rows.cu says what they are).
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace aien {

constexpr int F8_BLOCK = 128;
constexpr float F8_TOP = 448.0f, F8_LEAST = 1.17549435e-38f;      // the largest e4m3 number; 2^-126

__device__ __forceinline__ uint32_t f8_bits(float v) { return __float_as_uint(fabsf(v)); }
// m * (1 / 448): with the reciprocal's rounding and the product's at most 1.75 half steps of float32 from m / 448.
__device__ __forceinline__ float f8_scale(uint32_t top) {
    return top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fmaxf(__uint_as_float(top) * (1.0f / F8_TOP), F8_LEAST);
}
// One instruction of the special-function unit, at most a unit off, for ordinary numbers.
__device__ __forceinline__ float f8_reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// 1 / scale as float32 rounds it, so that a code is e4m3(x * (1 / scale)) to the bit: the instruction's result, corrected once by its exact residue (Markstein, 1990;
// compared with the rounded quotient over all mantissas at eight exponents).  A scale and its reciprocal are ordinary numbers, 2^-126 to 2^120.  Gated
// rows of 2,048 x 12,288 in 25.0 us, with a division 26.0.
__device__ __forceinline__ float f8_inverse(float scale) {
    const float r = f8_reciprocal(scale);
    return fmaf(fmaf(-scale, r, 1.0f), r, r);
}

// ---------------------------------------------------------------- gated activations
// One float32 number, or two in a pair of registers that one instruction takes.
__device__ __forceinline__ uint64_t f8_two(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(__float_as_uint(a)), "r"(__float_as_uint(b)));
    return v;
}
__device__ __forceinline__ float2 f8_split(uint64_t v) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float f8_ex2(float v) {
    float t;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(v));
    return t;
}
template <typename V> struct F8Math;
template <> struct F8Math<float> {
    using V = float;
    static __device__ __forceinline__ V all(float v) { return v; }
    static __device__ __forceinline__ V mul(V a, V b) { return __fmul_rn(a, b); }                        // (never one instruction with an addition)
    static __device__ __forceinline__ V add(V a, V b) { return __fadd_rn(a, b); }
    static __device__ __forceinline__ V mad(V a, V b, V c) { return fmaf(a, b, c); }
    static __device__ __forceinline__ V larger(V a, V b) { return fmaxf(a, b); }
    static __device__ __forceinline__ V minus_abs(V a, float least) { return fmaxf(-fabsf(a), least); }
    static __device__ __forceinline__ V ex2(V a) { return f8_ex2(a); }
    static __device__ __forceinline__ V minus_reciprocal(V a) { return f8_reciprocal(-a); }
};
template <> struct F8Math<uint64_t> {
    using V = uint64_t;
    static __device__ __forceinline__ V all(float v) { return f8_two(v, v); }
    static __device__ __forceinline__ V mul(V a, V b) { V r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
    static __device__ __forceinline__ V add(V a, V b) { V r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
    static __device__ __forceinline__ V mad(V a, V b, V c) { V r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
    template <typename F> static __device__ __forceinline__ V each(V a, F f) { const float2 x = f8_split(a); return f8_two(f(x.x), f(x.y)); }
    static __device__ __forceinline__ V larger(V a, V b) { const float2 x = f8_split(a), y = f8_split(b); return f8_two(fmaxf(x.x, y.x), fmaxf(x.y, y.y)); }
    static __device__ __forceinline__ V minus_abs(V a, float least) { return each(a, [=](float v) { return fmaxf(-fabsf(v), least); }); }
    static __device__ __forceinline__ V ex2(V a) { return each(a, [](float v) { return f8_ex2(v); }); }
    static __device__ __forceinline__ V minus_reciprocal(V a) { return each(a, [](float v) { return f8_reciprocal(-v); }); }
};
// -g / (1 + exp(-x)), x of g's sign: -max(g, g e) / (1 + e) with e = exp(-|x|), so that the divisor lies between 1 and 2 and a small result is as exact as
// a large one.  e is 2^p times a correction by what p = -|x| log2(e), rounded, lacks (rest: |x| 2^-24 at the most, which the instruction
// alone would be off by, relatively); it is made 2^24 times as large, so that the instruction's flush of small numbers to 0 stays below |x| = 103, where e leaves
// float32.  Adding 24 to p rounds it again; taking 24 off the sum again is exact.  The quotient is a product with an approximate reciprocal, corrected
// by its exact residue (Markstein, 1990): next to always the rounded quotient.  In all 9 half steps of float32 at the most, beside what x is off.  Gated rows of
// 2,048 x 12,288 in 25.0 us; with expf and a division 33.6, with the two instructions alone, off by 1.2 |x| half steps, 23.8.
// (The sign is the reciprocal's, whose operand may be negated; the residue is then one product with the divisor as it is.)
template <typename V>
__device__ __forceinline__ V f8_minus_logistic(V g, V x) {
    using F = F8Math<V>;
    const V a = F::minus_abs(x, -200.0f), up = F::add(F::mul(a, F::all(1.44269504f)), F::all(24.0f)), p = F::add(up, F::all(-24.0f));
    const V rest = F::mad(p, F::all(1.90465430e-9f), F::mad(p, F::all(-0.693147182f), a));              // a - p ln 2, ln 2 in two parts
    const V t = F::ex2(up), e = F::mad(t, rest, t), d = F::mad(e, F::all(0x1p-24f), F::all(1.0f));
    const V n = F::larger(g, F::mul(F::mul(g, e), F::all(0x1p-24f))), r = F::minus_reciprocal(d), q = F::mul(n, r);
    return F::mad(F::mad(q, d, n), r, q);
}
// -act(g) * u: silu, or the gelu in its tanh form, 0.5 g (1 + tanh z) = g / (1 + exp(-2 z)) with z = sqrt(2 / pi) (g + 0.044715 g^3).  (As 1 + tanh z nothing
// would be left of it for gates below -5.)
template <bool GELU, typename V>
__device__ __forceinline__ V f8_minus_gate(V g, V u) {
    using F = F8Math<V>;
    V x = g;
    if (GELU) x = F::mul(g, F::mad(F::mul(g, g), F::all(0.0713548163f), F::all(1.59576912f)));           // 2 z
    return F::mul(f8_minus_logistic<V>(g, x), u);
}
__device__ __forceinline__ uint32_t f8_pair(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 f8_pack(const float v[8], float inv) {
    return make_uint2(f8_pair(v[0] * inv, v[1] * inv) | f8_pair(v[2] * inv, v[3] * inv) << 16,
                      f8_pair(v[4] * inv, v[5] * inv) | f8_pair(v[6] * inv, v[7] * inv) << 16);
}

}  // namespace aien
