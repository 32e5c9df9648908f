// Epilogue arithmetic shared by the 8-bit integer kernels.
//
// Activations of f32 results are computed with the full-precision functions;
// 16-bit results take forms of two MUFU operations whose error is below their
// rounding.
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
