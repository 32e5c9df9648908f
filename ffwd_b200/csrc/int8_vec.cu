// 8-bit integer projections of a few rows (see int8.cuh): the weights are read
// once, straight from memory into registers, and multiplied with the rows by
// the four-way byte dot product.  Bound by the weights' bytes; a tensor-core
// tile would spend its rows' work on at most 4.  One row of 4096 x 12288: 8.5 us
// (weights in L2), of gate and up of 4096 x 1024: 2.6 us, of 24 + 8 heads, K =
// 1024: 3.5 us.
//
// A warp takes R weight rows, a lane 16 bytes of each at a time (512 bytes of
// a row per load), all of the rows' sums stay in registers (R x MT integers)
// and meet in one warp-wide integer add each.  The head form gives a block a
// whole head, whose values meet in shared memory for the norm and rotation.
#include "host_util.h"
#include "int8.cuh"
#include "int8_epi.cuh"
#include "launch_util.cuh"
#include "ptx.cuh"

namespace fb {
namespace {

__device__ __forceinline__ uint4 ldg16(const int8_t *p) {
    return ld_global(reinterpret_cast<const uint4 *>(p));
}

// Bytes of chunk [k, k + 16) at or past K cleared (weights and rows may hold
// anything in their padding; one zero factor is enough).
__device__ __forceinline__ uint4 clip16(uint4 v, int k, int K) {
    if (k + 16 <= K) return v;
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = K - k - 4 * i;
        if (left <= 0) w[i] = 0;
        else if (left < 4) w[i] &= (1u << (8 * left)) - 1u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ int dot16(uint4 a, uint4 b, int c) {
    c = __dp4a((int)a.x, (int)b.x, c);
    c = __dp4a((int)a.y, (int)b.y, c);
    c = __dp4a((int)a.z, (int)b.z, c);
    return __dp4a((int)a.w, (int)b.w, c);
}

// acc[r][m] = sum over k of w[r][k] x[m][k], complete in every lane.  Rows m
// at or past M read row M - 1 (their sums are not used).
template <int R, int MT>
__device__ __forceinline__ void dots(const int8_t *const (&w)[R], const I8Params &p, int lane,
                                     int (&acc)[R][MT]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[r][m] = 0;
    const int8_t *x[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = p.x + (size_t)min(m, p.M - 1) * p.ldx;
    constexpr int U = R >= 4 ? 2 : 4;  // loads of a row in flight
    int k = lane * 16;
    for (; k + (U - 1) * 512 < p.K; k += U * 512) {
        uint4 wv[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) wv[u][r] = ldg16(w[r] + k + u * 512);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const uint4 xv = clip16(ldg16(x[m] + k + u * 512), k + u * 512, p.K);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r][m] = dot16(wv[u][r], xv, acc[r][m]);
            }
    }
    for (; k < p.K; k += 512) {
        uint4 wv[R];
#pragma unroll
        for (int r = 0; r < R; ++r) wv[r] = ldg16(w[r] + k);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint4 xv = clip16(ldg16(x[m] + k), k, p.K);
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][m] = dot16(wv[r], xv, acc[r][m]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[r][m] = __reduce_add_sync(0xffffffffu, acc[r][m]);
}

// acc[r][m] of this lane's (r, m) = (lane / MT, lane % MT).
template <int R, int MT>
__device__ __forceinline__ int mine(const int (&acc)[R][MT], int lane) {
    int v = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m)
            if (lane == r * MT + m) v = acc[r][m];
    return v;
}

__device__ __forceinline__ float scaled(int acc, float s, const float *ws, const float *bias,
                                        int n) {
    return fmaf((float)acc * s, ld_global(ws + n), bias ? ld_global(bias + n) : 0.0f);
}

// The first 2 KB of a row on their way to L2; before the wait for the stream's
// previous kernel (as a rule the one that quantises the rows).
__device__ __forceinline__ void prefetch_row(const int8_t *w, int K, int lane) {
    if (lane * 128 < min(K, 2048))
        asm volatile("prefetch.global.L2 [%0];" ::"l"(w + lane * 128));
}

constexpr int kWarps = 4;

template <int R, int MT>
__global__ void __launch_bounds__(kWarps * 32) vec_store_kernel(const I8Params p) {
    const int lane = threadIdx.x & 31;
    const int n0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * R;
    const int8_t *w[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        w[r] = p.w + (size_t)min(n0 + r, p.N - 1) * p.ldw;
        prefetch_row(w[r], p.K, lane);
    }
    griddep_wait();
    griddep_launch();
    if (n0 >= p.N) return;
    int acc[R][MT];
    dots<R, MT>(w, p, lane, acc);
    const int a = mine<R, MT>(acc, lane);
    const int n = n0 + lane / MT, m = lane % MT;
    if (lane < R * MT && n < p.N && m < p.M)
        i8::store1(p.y, p.type, (size_t)m * p.ldy + n,
                   i8::act1(scaled(a, ld_global(p.xs + m), p.ws, p.bias, n), p.act), p.accumulate);
}

// R columns of gate and up each.
template <int R, int MT>
__global__ void __launch_bounds__(kWarps * 32) vec_gated_kernel(const I8Params p) {
    const int lane = threadIdx.x & 31;
    const int n0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * R;
    const int8_t *w[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        w[r] = p.w + (size_t)min(n0 + r, p.N - 1) * p.ldw;
        w[R + r] = p.w2 + (size_t)min(n0 + r, p.N - 1) * p.ldw2;
        prefetch_row(w[r], p.K, lane);
        prefetch_row(w[R + r], p.K, lane);
    }
    griddep_wait();
    griddep_launch();
    if (n0 >= p.N) return;
    int acc[2 * R][MT];
    dots<2 * R, MT>(w, p, lane, acc);
    const int v = mine<2 * R, MT>(acc, lane);
    const int up = __shfl_down_sync(0xffffffffu, v, R * MT);
    const int n = n0 + lane / MT, m = lane % MT;
    if (lane < R * MT && n < p.N && m < p.M) {
        const float s = ld_global(p.xs + m);
        const float g = i8::act1(scaled(v, s, p.ws, p.bias, n), p.act);
        i8::store1(p.y, p.type, (size_t)m * p.ldy + n, g * scaled(up, s, p.ws2, p.bias2, n), 0);
    }
}

constexpr int kHeadWarps = 16;

template <int HD, int MT>
__global__ void __launch_bounds__(kHeadWarps * 32) vec_heads_kernel(const I8Params p) {
    __shared__ float v[MT][HD];
    constexpr int R = 4, HALF = HD / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x;
    for (int e0 = warp * R; e0 < HD; e0 += kHeadWarps * R)
        for (int r = 0; r < R; ++r)
            prefetch_row(p.w + (size_t)(head * HD + e0 + r) * p.ldw, p.K, lane);
    griddep_wait();
    griddep_launch();
    for (int e0 = warp * R; e0 < HD; e0 += kHeadWarps * R) {
        const int n0 = head * HD + e0;
        const int8_t *w[R];
#pragma unroll
        for (int r = 0; r < R; ++r) w[r] = p.w + (size_t)(n0 + r) * p.ldw;
        int acc[R][MT];
        dots<R, MT>(w, p, lane, acc);
        const int a = mine<R, MT>(acc, lane);
        const int r = lane / MT, m = lane % MT;
        if (lane < R * MT)
            v[m][e0 + r] = m < p.M ? scaled(a, ld_global(p.xs + m), p.ws, p.bias, n0 + r) : 0.0f;
    }
    __syncthreads();
    const int m = warp;  // one warp per row
    if (m >= MT || m >= p.M) return;
    float a[HALF / 32], b[HALF / 32];
#pragma unroll
    for (int j = 0; j < HALF / 32; ++j) {
        a[j] = v[m][lane + 32 * j];
        b[j] = v[m][HALF + lane + 32 * j];
    }
    if (head < p.n_q_heads + p.n_kv_heads) {
        const float *nw = head < p.n_q_heads ? p.q_norm : p.k_norm;
        const int ps = ld_global(p.pos + m);
        const bool bad = ps < 0 || ps >= p.n_pos;
        if (bad && lane == 0) set_error(p.err, kErrBadPosition);
        float inv = bad ? i8::nan_f() : 1.0f;
        if (nw) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < HALF / 32; ++j) ss += a[j] * a[j] + b[j] * b[j];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv *= 1.0f / sqrtf(ss / (float)HD + p.eps);
        }
        const size_t t = (size_t)(bad ? 0 : ps) * HALF;
#pragma unroll
        for (int j = 0; j < HALF / 32; ++j) {
            const int e = lane + 32 * j;
            const float c = ld_global(p.cos + t + e), s = ld_global(p.sin + t + e);
            const float x1 = a[j] * inv * (nw ? ld_global(nw + e) : 1.0f);
            const float x2 = b[j] * inv * (nw ? ld_global(nw + HALF + e) : 1.0f);
            a[j] = i8::rotate(x1, x2, c, s, -1.0f);
            b[j] = i8::rotate(x2, x1, c, s, 1.0f);
        }
    }
    const size_t o = (size_t)m * p.ldy + (size_t)head * HD;
#pragma unroll
    for (int j = 0; j < HALF / 32; ++j) {
        i8::store1(p.y, p.type, o + lane + 32 * j, a[j], 0);
        i8::store1(p.y, p.type, o + HALF + lane + 32 * j, b[j], 0);
    }
}

template <int R, int MT>
cudaError_t run_store(const I8Params &p, cudaStream_t st) {
    return launch_k(vec_store_kernel<R, MT>, dim3((p.N + kWarps * R - 1) / (kWarps * R)),
                    dim3(kWarps * 32), 0, st, p);
}

template <int R, int MT>
cudaError_t run_gated(const I8Params &p, cudaStream_t st) {
    return launch_k(vec_gated_kernel<R, MT>, dim3((p.N + kWarps * R - 1) / (kWarps * R)),
                    dim3(kWarps * 32), 0, st, p);
}

// More weight rows per warp once there are enough of them to fill the SMs'
// warps, and with more quantised rows: a warp's loads of those are shared among
// its weight rows.
template <int MT>
cudaError_t run(int epi, const I8Params &p, int num_sms, cudaStream_t st) {
    const int warps = num_sms * 16;
    switch (epi) {
    case kI8Store:
        if (MT == 4 || p.N >= 4 * warps) return run_store<4, MT>(p, st);
        if constexpr (MT == 1) {
            if (p.N < 2 * warps) return run_store<1, MT>(p, st);
        }
        if constexpr (MT <= 2) return run_store<2, MT>(p, st);
        break;
    case kI8Gated:
        if (MT == 4 || p.N >= 2 * warps) return run_gated<2, MT>(p, st);
        if constexpr (MT <= 2) return run_gated<1, MT>(p, st);
        break;
    case kI8Heads: {
        const int heads = p.n_q_heads + 2 * p.n_kv_heads;
        return p.head_dim == 128 ? launch_k(vec_heads_kernel<128, MT>, dim3(heads),
                                            dim3(kHeadWarps * 32), 0, st, p)
                                 : launch_k(vec_heads_kernel<64, MT>, dim3(heads),
                                            dim3(kHeadWarps * 32), 0, st, p);
    }
    }
    return cudaErrorInvalidValue;
}

}  // namespace

// Up to 2 rows; 3 and 4 while K and the weights are small (4 rows of 8192 x 1024
// 3.9 us against 5.5 of int8_mid.cu, of 1024 x 2048 4.5 and 5.3; of 1024 x 4096
// 7.7 and 6.3, of 4096 x 12288 21 and 10.9; of 24 + 8 heads, K = 1024 6.2 and 7.0,
// K = 2048 8.8 and 7.5).
bool i8_vec_fits(int epi, const I8Params &p) {
    if (p.M <= 2) return true;
    return p.M <= 4 && p.K <= (epi == kI8Heads ? 1024 : 2048) &&
           (long long)p.N * p.K * (epi == kI8Gated ? 2 : 1) <= 16 << 20;
}

int i8_vec_launch(int epi, const I8Params &p, int num_sms, cudaStream_t stream) {
    if (p.M <= 1) return run<1>(epi, p, num_sms, stream);
    if (p.M <= 2) return run<2>(epi, p, num_sms, stream);
    return run<4>(epi, p, num_sms, stream);
}

}  // namespace fb
