// Epilogue arithmetic shared by the 8-bit integer kernels.
//
// Activations of f32 results are computed with the full-precision functions;
// 16-bit results take forms of two MUFU operations whose error (a few 2^-24 of
// the argument) is far below their rounding: the epilogue shares the SM with a
// tile's products (4096 cycles at K = 1024), which erff for its 32768 values
// alone would pass (8192 x 4096 x 1024 rows with GELU: 88 us with erff).
#pragma once

#include "gemm_epi.cuh"
#include "int8.cuh"
#include "ptx.cuh"

namespace fb {
namespace i8 {

__device__ __forceinline__ float act_full(float x, int act) {
    switch (act) {
    case kI8Silu: return x / (1.0f + expf(-x));
    case kI8GeluErf: return epi::gelu_erf(x);
    case kI8GeluTanh: return epi::gelu_tanh(x);
    }
    return x;
}

// GELU by the normal distribution's upper tail, h = (1 - erf(z)) / 2 at z = |x| /
// sqrt 2, as x h or x - x h.  1 - erf(z) = t (a1 + t (a2 + ... + t a5)) e^(-z^2),
// t = 1 / (1 + p z): Abramowitz and Stegun, 7.1.26, off by at most 1.5e-7.
__device__ __forceinline__ float gelu_erf_16(float x) {
    const float ax = fabsf(x);
    const float t = __fdividef(1.0f, fmaf(0.3275911f * 0.70710678f, ax, 1.0f));
    float a = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
    a = fmaf(a, t, 0.5f * 1.421413741f);
    a = fmaf(a, t, 0.5f * -0.284496736f);
    a = fmaf(a, t, 0.5f * 0.254829592f);
    // e^(-x^2 / 2) as a power of two.
    const float h = a * t * ex2_approx(x * x * -0.72134752f);
    const float xh = ax * h;
    return x > 0.0f ? x - xh : -xh;
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
