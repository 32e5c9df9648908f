// Projections in 8-bit integers: rows quantised with one scale each, weights
// with one scale per output channel, products summed exactly in 32-bit
// integers, scales and the layer's elementwise work in the epilogue.
//
//   q[m, k] = rint(x[m, k] / s[m]),  s[m] = max_k |x[m, k]| / 127
//   y[m, n] = (sum_k q[m, k] p[n, k]) * s[m] * t[n] + b[n]
//
// The integer sums do not depend on their order, so every variant and tile
// shape gives the same bits up to the epilogue's f32 arithmetic.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace fb {

// Element types of rows and results.
enum I8Type : int { kI8F32 = 0, kI8BF16 = 1, kI8F16 = 2 };

enum I8Act : int { kI8None = 0, kI8Silu = 1, kI8GeluErf = 2, kI8GeluTanh = 3 };

enum I8Epi : int {
    kI8Store = 0,  // y = act(acc * s * t + b), or y += it
    kI8Gated = 1,  // y = act(gate) * up
    kI8Heads = 2,  // per-head RMSNorm (q and k heads) + NeoX RoPE
};

// int8 is exact in 32-bit sums up to this many products of at most 2^14 each.
constexpr int kI8MaxK = 131071;

struct I8Params {
    int M, N, K;  // kI8Gated: N columns of gate and as many of up
    const int8_t *x;
    long long ldx;
    const float *xs;  // [M]
    const int8_t *w;  // [N, K] (kI8Gated: gate)
    const int8_t *w2;  // up
    long long ldw, ldw2;
    const float *ws, *ws2;      // [N]
    const float *bias, *bias2;  // [N] or null
    void *y;
    int type;  // I8Type of y
    long long ldy;
    int act;
    int accumulate;  // f32 y: y += result
    // kI8Heads
    int n_q_heads, n_kv_heads, head_dim, n_pos;
    const int *pos;          // [M]
    const float *cos, *sin;  // [n_pos, head_dim / 2]
    const float *q_norm, *k_norm;  // [head_dim] or null
    float eps;
    int *err;  // device error word or null
};

// x [M, K] of `type` (row stride ldx elements) -> q int8 [M, K] (row stride
// ldq, a multiple of 16) and s [M]; with `norm`, of x * norm / rms(x) instead.
// A row of zeros has s = 0; a row whose values (or products with norm, or sum of
// squares) are not finite has s = NaN and q = 0.  Returns a cudaError_t value.
int i8_quantize_launch(const void *x, int type, long long ldx, const float *norm, float eps,
                       int8_t *q, long long ldq, float *s, int M, int K, int num_sms,
                       cudaStream_t stream);

// LayerNorm of x [M, K] f32 in place (row stride K) with the rows' codes and
// scales beside it; for the widths that fit (at most 1024, multiples of 16).
// A row that is not finite, or below 1e-30 throughout, gets zeros.
bool i8_layernorm_quantize_fits(int K);
int i8_layernorm_quantize_launch(float *x, const float *gamma, const float *beta, float eps,
                                 int8_t *q, float *s, int M, int K, int num_sms,
                                 cudaStream_t stream);

// Whether the streaming kernel for few rows (int8_vec.cu) takes this product.
bool i8_vec_fits(int epi, const I8Params &p);
int i8_vec_launch(int epi, const I8Params &p, int num_sms, cudaStream_t stream);

// Kernel for a few tens of rows (int8_mid.cu): likewise; -1 with a message, or 0.
bool i8_mid_fits(int epi, const I8Params &p, int num_sms);
int i8_mid_run(int epi, const I8Params &p, int num_sms, cudaStream_t stream);

// Tensor-core kernel (int8_gemm.cu).  -1 with a message, or 0.
int i8_gemm_run(int epi, const I8Params &p, int num_sms, cudaStream_t stream);

// Either kernel, by size; -1 with a message, or 0.
int i8_project(int epi, const I8Params &p, int num_sms, cudaStream_t stream);

}  // namespace fb
