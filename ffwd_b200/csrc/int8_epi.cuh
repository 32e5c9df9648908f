// Epilogue arithmetic shared by the 8-bit integer kernels.
//
// Activations work on pairs of values in packed f32 arithmetic with two
// special-function operations each (a power of two and a reciprocal), for every
// output type: the epilogue shares the SM with the next tile's products (4096
// cycles at K = 1024 for 32768 values), and the library's erff, tanhf and expf
// in one kernel outgrow the instruction cache as well (8192 x 4096 x 1024 with
// GELU: 64 us).
#pragma once

#include "int8.cuh"
#include "ptx.cuh"

namespace fb {
namespace i8 {

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float2 both(float c) { return make_float2(c, c); }

// GELU of two values by the normal distribution's upper tail, h = (1 - erf(z)) / 2
// at z = |x| / sqrt 2, as max(x, 0) - |x| h.  1 - erf(z) = P(t) e^(-z^2) with t =
// 1 / (1 + 0.4 z) and P of degree 6 without a constant, fitted here (weighted
// least squares in t, z <= 7): x h is off by at most 2e-8 plus rounding.
__device__ __forceinline__ float2 gelu_erf(float2 x) {
    // (finite, so that an infinite x gives itself or 0)
    const float2 ax = make_float2(fminf(fabsf(x.x), 3.4e38f), fminf(fabsf(x.y), 3.4e38f));
    const float2 den = fma_f32x2(ax, both(0.28284271f), both(1.0f));
    const float2 t = make_float2(rcp_approx(den.x), rcp_approx(den.y));
    float2 a = fma_f32x2(t, both(0.5f * -0.20369884f), both(0.5f * 0.7232648f));
    a = fma_f32x2(a, t, both(0.5f * -0.3939358f));
    a = fma_f32x2(a, t, both(0.5f * 0.48692873f));
    a = fma_f32x2(a, t, both(0.5f * 0.15432052f));
    a = fma_f32x2(a, t, both(0.5f * 0.23312044f));
    // e^(-x^2 / 2) as a power of two.
    const float2 e = mul_f32x2(mul_f32x2(x, both(-0.72134752f)), x);
    const float2 h = mul_f32x2(mul_f32x2(a, t), make_float2(ex2_approx(e.x), ex2_approx(e.y)));
    return fma_f32x2(make_float2(-ax.x, -ax.y), h, make_float2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
}

// x / (1 + d) of two values.
__device__ __forceinline__ float2 over_1p(float2 x, float2 d) {
    d = add_f32x2(d, both(1.0f));
    return mul_f32x2(x, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
}

// SiLU, x / (1 + 2^e), e = -x log2(e): e in two parts (its rounding alone would
// be off by |x| 2^-24 of the result for negative x).
__device__ __forceinline__ float2 silu(float2 x) {
    // (beyond 200 the result is x or 0, and the parts would pass f32)
    const float2 c = make_float2(fminf(fmaxf(x.x, -200.0f), 200.0f),
                                 fminf(fmaxf(x.y, -200.0f), 200.0f));
    const float2 e = mul_f32x2(c, both(-1.44269504f));
    const float2 ne = make_float2(-e.x, -e.y);
    const float2 lo = fma_f32x2(c, both(-1.92596299e-8f), fma_f32x2(c, both(-1.44269504f), ne));
    const float2 w = make_float2(ex2_approx(e.x), ex2_approx(e.y));
    // (an infinite power times a lo of zero would be NaN)
    const float2 wf = make_float2(fminf(w.x, 3.0e38f), fminf(w.y, 3.0e38f));
    return over_1p(x, fma_f32x2(wf, mul_f32x2(lo, both(0.69314718f)), w));
}

// GELU, tanh form: 0.5 (1 + tanh(v)) = 1 / (1 + 2^e), v = sqrt(2 / pi) (x +
// 0.044715 x^3), e = -2 log2(e) v.
__device__ __forceinline__ float2 gelu_tanh(float2 x) {
    const float2 k = fma_f32x2(mul_f32x2(x, x), both(-0.10294324f), both(-2.3022082f));
    const float2 e = mul_f32x2(x, k);
    return over_1p(x, make_float2(ex2_approx(e.x), ex2_approx(e.y)));
}

__device__ __forceinline__ float2 act2(float2 x, int act) {
    switch (act) {
    case kI8Silu: return silu(x);
    case kI8GeluErf: return gelu_erf(x);
    case kI8GeluTanh: return gelu_tanh(x);
    }
    return x;
}

__device__ __forceinline__ float act1(float x, int act) { return act2(make_float2(x, x), act).x; }

// A value z rotated with its head's other half o: z c -+ o s (- in the first half,
// where sign is -1), rounded alike in every kernel.
__device__ __forceinline__ float rotate(float z, float o, float c, float s, float sign) {
    return fmaf(sign * o, s, __fmul_rn(z, c));
}

__device__ __forceinline__ float nan_f() { return __uint_as_float(0x7FC00000u); }

__device__ __forceinline__ uint16_t to_16(float v, int type) {
    return type == kI8BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v))
                           : __half_as_ushort(__float2half_rn(v));
}

__device__ __forceinline__ void store1(void *y, int type, size_t off, float v, int accumulate) {
    if (type == kI8F32) {
        float *o = static_cast<float *>(y) + off;
        *o = accumulate ? *o + v : v;
    } else {
        static_cast<uint16_t *>(y)[off] = to_16(v, type);
    }
}

}  // namespace i8
}  // namespace fb
