// Rows to 8-bit integers with one scale each (see int8.cuh), optionally after
// an RMSNorm.  Bound by memory: each row is read once into registers (rows of
// up to 16384 columns; longer ones are read twice) and written once at a byte
// per value.
//
// Rounding.  The code of a value is the nearest integer of v / s (s = amax / 127,
// both quotients in f64; ties to even).  In f32 the
// quotient is off by a few units in the last place (the product x * norm, the
// reciprocal and the product with it: 4 x 2^-24 x 127 < 4e-5), which matters
// only next to the border of two codes; there, about one value in 10^4, it is
// taken again in f64.  The row's RMS cancels out of v / s, so with `norm` the
// codes depend on x * norm alone and only the scale carries the RMS.
#include "int8.cuh"
#include "launch_util.cuh"
#include "ptx.cuh"

namespace fb {
namespace {

constexpr float kTieBand = 4e-5f;

template <int TYPE>
__device__ __forceinline__ float load1(const void *x, size_t i) {
    if (TYPE == kI8F32) return static_cast<const float *>(x)[i];
    const uint16_t h = static_cast<const uint16_t *>(x)[i];
    if (TYPE == kI8BF16) return __uint_as_float((uint32_t)h << 16);
    return __half2float(__ushort_as_half(h));
}

// Columns [c, c + 8) of the row at x; columns at or past K read as 0.
template <int TYPE>
__device__ __forceinline__ void load8(const void *x, size_t off, int c, int K, bool vec,
                                      float (&v)[8]) {
    if (vec && c + 8 <= K) {
        if (TYPE == kI8F32) {
            const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(x) + off + c);
            const float4 a = __ldg(p), b = __ldg(p + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(
                static_cast<const uint16_t *>(x) + off + c));
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (TYPE == kI8BF16) {
                    v[2 * i] = __uint_as_float(w[i] << 16);
                    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                    v[2 * i] = f.x;
                    v[2 * i + 1] = f.y;
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? load1<TYPE>(x, off + c + i) : 0.0f;
}

__device__ __forceinline__ void load8_norm(const float *w, int c, int K, bool vec, float (&g)[8]) {
    load8<kI8F32>(w, 0, c, K, vec, g);
}

// The residue of the f32 product x * w = p (exact unless it underflows).
__device__ __forceinline__ float residue(float x, float w, float p) { return fmaf(x, w, -p); }

// max(m, |v|), NaN if either is.
__device__ __forceinline__ float max_abs(float m, float v) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
    return r;
}

// 1.5 x 2^23: adding it leaves the nearest integer in the low bits of the sum
// (ties to even), two's complement in the lowest byte.
constexpr float kRound = 12582912.0f;

__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
    const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}

// Codes of eight values (p = x, or x * g with a norm) of a row whose largest
// magnitude is amax + amax_lo; written as 8 bytes, or as fewer at the row's end.
template <bool NORM>
__device__ __forceinline__ void put8(const float (&x)[8], const float (&g)[8], float inv,
                                     float amax, float amax_lo, int8_t *q, int c, int K) {
    float code[8];
    float far = 0.0f;  // largest distance from a code
    const float2 inv2 = make_float2(inv, inv), up = make_float2(kRound, kRound),
                 down = make_float2(-kRound, -kRound);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 t = make_float2(x[2 * i], x[2 * i + 1]);
        if (NORM) t = mul_f32x2(t, make_float2(g[2 * i], g[2 * i + 1]));
        t = mul_f32x2(t, inv2);
        const float2 f = add_f32x2(t, up);
        const float2 d = add_f32x2(t, mul_f32x2(add_f32x2(f, down), make_float2(-1.0f, -1.0f)));
        far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
        code[2 * i] = f.x;
        code[2 * i + 1] = f.y;
    }
    uint32_t w0 = low_bytes(code[0], code[1], code[2], code[3]);
    uint32_t w1 = low_bytes(code[4], code[5], code[6], code[7]);
    if (far > 0.5f - kTieBand) {
        // In f64, one value after another (a rare path, kept small).
        const double s = ((double)amax + (double)amax_lo) / 127.0;
        uint32_t near = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = (NORM ? x[i] * g[i] : x[i]) * inv - (code[i] - kRound);
            near |= (fabsf(d) > 0.5f - 2.0f * kTieBand ? 1u : 0u) << i;
        }
#pragma unroll 1
        for (; near; near &= near - 1) {
            const int j = __ffs(near) - 1;
            float xj = x[0], gj = g[0];
#pragma unroll
            for (int i = 1; i < 8; ++i)
                if (i == j) {
                    xj = x[i];
                    if (NORM) gj = g[i];
                }
            const double v = NORM ? (double)xj * (double)gj : (double)xj;
            const uint32_t byte = (uint32_t)(int)rint(v / s) & 0xFF;
            const int sh = 8 * (j & 3);
            const uint32_t w = ((j < 4 ? w0 : w1) & ~(0xFFu << sh)) | byte << sh;
            if (j < 4) w0 = w;
            else w1 = w;
        }
    }
    if (c + 8 <= K) {
        *reinterpret_cast<uint2 *>(q + c) = make_uint2(w0, w1);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < K) q[c + i] = (int8_t)((i < 4 ? w0 : w1) >> (8 * (i & 3)));
    }
}

// W warps per row, each thread holding NV groups of 8 columns (NV = 0: any
// width, the row read again for the second pass).  A block of max(W, 8) warps.
template <int TYPE, bool NORM, int W, int NV>
__global__ void __launch_bounds__((W > 8 ? W : 8) * 32)
    quantize_kernel(const void *x, long long ldx, const float *norm, float eps, int8_t *q,
                    long long ldq, float *s, int M, int K, int vec_x, int vec_n) {
    constexpr int NW = W > 8 ? W : 8;
    __shared__ uint32_t sh_max[NW];
    __shared__ float sh_sum[NW], sh_lo[NW];
    griddep_wait();
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int wr = warp % W;  // warp of the row
    const int row = blockIdx.x * (NW / W) + warp / W;
    const bool live = row < M;
    if (W == 1 && !live) return;
    const size_t off = live ? (size_t)row * ldx : 0;
    const int t = wr * 32 + lane;
    constexpr int NR = NV > 0 ? NV : 1;
    float v[NR][8], g[NR][8];
    float mv = 0.0f;
    float ss = 0.0f;
    auto stats = [&](const float(&a)[8], const float(&b)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (NORM) ss = fmaf(a[i], a[i], ss);
            mv = max_abs(mv, NORM ? a[i] * b[i] : a[i]);
        }
    };
    if (live) {
        if (NV > 0) {
#pragma unroll
            for (int k = 0; k < NR; ++k) {
                const int c = (k * W * 32 + t) * 8;
                load8<TYPE>(x, off, c, K, vec_x, v[k]);
                if (NORM) load8_norm(norm, c, K, vec_n, g[k]);
            }
#pragma unroll
            for (int k = 0; k < NR; ++k) stats(v[k], g[k]);
        } else {
            for (int c = t * 8; c < K; c += W * 256) {
                load8<TYPE>(x, off, c, K, vec_x, v[0]);
                if (NORM) load8_norm(norm, c, K, vec_n, g[0]);
                stats(v[0], g[0]);
            }
        }
    }
    // Magnitudes compare as unsigned integers, NaN above infinity.
    const uint32_t mine = __float_as_uint(mv);
    uint32_t mx = __reduce_max_sync(0xffffffffu, mine);
    if (NORM) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    if (W > 1) {
        if (lane == 0) {
            sh_max[warp] = mx;
            if (NORM) sh_sum[warp] = ss;
        }
        __syncthreads();
        const int w0 = warp - wr;
        mx = 0;
        ss = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            mx = max(mx, sh_max[w0 + i]);
            if (NORM) ss += sh_sum[w0 + i];
        }
    }
    const float amax = __uint_as_float(mx);
    float amax_lo = 0.0f;
    if (NORM) {
        // The largest product in full: among the values whose rounded product
        // is the maximum, the largest residue (rounding keeps the order).
        float lo = -INFINITY;
        auto resid = [&](const float(&a)[8], const float(&b)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = a[i] * b[i];
                if (fabsf(p) == amax) {
                    const float e = residue(a[i], b[i], p);
                    lo = fmaxf(lo, p < 0.0f ? -e : e);
                }
            }
        };
        if (live && mine == mx) {
            if (NV > 0) {
#pragma unroll
                for (int k = 0; k < NR; ++k) resid(v[k], g[k]);
            } else {
                for (int c = t * 8; c < K; c += W * 256) {
                    load8<TYPE>(x, off, c, K, vec_x, v[0]);
                    load8_norm(norm, c, K, vec_n, g[0]);
                    resid(v[0], g[0]);
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lo = fmaxf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        if (W > 1) {
            if (lane == 0) sh_lo[warp] = lo;
            __syncthreads();
            const int w0 = warp - wr;
            lo = sh_lo[w0];
#pragma unroll
            for (int i = 1; i < W; ++i) lo = fmaxf(lo, sh_lo[w0 + i]);
        }
        amax_lo = lo;
    }
    if (!live) return;
    const bool finite = mx < 0x7F800000u && (!NORM || ss < INFINITY);
    int8_t *qr = q + (size_t)row * ldq;
    if (!finite || mx == 0) {
        if (t == 0) s[row] = finite ? 0.0f : __uint_as_float(0x7FC00000u);
        for (int c = t * 8; c < K; c += W * 256) {
            if (c + 8 <= K)
                *reinterpret_cast<uint2 *>(qr + c) = make_uint2(0, 0);
            else
                for (int i = c; i < K; ++i) qr[i] = 0;
        }
        return;
    }
    if (t == 0) {
        double sc = ((double)amax + (double)amax_lo) / 127.0;
        if (NORM) sc /= sqrt((double)ss / (double)K + (double)eps);
        s[row] = (float)sc;
    }
    if (amax < 1e-30f) {
        // 127 / amax may pass f32: such rows go through f64, a value at a time.
        const double sc = ((double)amax + (double)amax_lo) / 127.0;
        for (int c = t; c < K; c += W * 32) {
            double v = (double)load1<TYPE>(x, off + c);
            if (NORM) v *= (double)norm[c];
            qr[c] = (int8_t)(int)rint(v / sc);
        }
        return;
    }
    const float inv = 127.0f / amax;
    if (NV > 0) {
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int c = (k * W * 32 + t) * 8;
            if (c < K) put8<NORM>(v[k], g[k], inv, amax, amax_lo, qr, c, K);
        }
    } else {
        for (int c = t * 8; c < K; c += W * 256) {
            load8<TYPE>(x, off, c, K, vec_x, v[0]);
            if (NORM) load8_norm(norm, c, K, vec_n, g[0]);
            put8<NORM>(v[0], g[0], inv, amax, amax_lo, qr, c, K);
        }
    }
}

struct Args {
    const void *x;
    long long ldx;
    const float *norm;
    float eps;
    int8_t *q;
    long long ldq;
    float *s;
    int M, K, vec_x, vec_n;
};

template <int TYPE, bool NORM, int W, int NV>
cudaError_t run(const Args &a, cudaStream_t st) {
    constexpr int NW = W > 8 ? W : 8, R = NW / W;
    return launch_k(quantize_kernel<TYPE, NORM, W, NV>, dim3((a.M + R - 1) / R), dim3(NW * 32), 0,
                    st, a.x, a.ldx, a.norm, a.eps, a.q, a.ldq, a.s, a.M, a.K, a.vec_x, a.vec_n);
}

// Many rows: as few warps per row as hold it (a warp's own reductions, no
// block barrier).  Few rows (under two per SM): more warps per row, so that a
// row's loads are all in flight at once.
template <int TYPE, bool NORM>
cudaError_t pick(const Args &a, bool few, cudaStream_t st) {
    if (a.K <= 256) return run<TYPE, NORM, 1, 1>(a, st);
    if (!few) {
        if (a.K <= 512) return run<TYPE, NORM, 1, 2>(a, st);
        if (a.K <= 1024) return run<TYPE, NORM, 1, 4>(a, st);
    }
    if (a.K <= 1024) return run<TYPE, NORM, 4, 1>(a, st);
    if (!few) {
        if (a.K <= 2048) return run<TYPE, NORM, 4, 2>(a, st);
        if (a.K <= 4096) return run<TYPE, NORM, 4, 4>(a, st);
    }
    if (a.K <= 4096) return run<TYPE, NORM, 16, 1>(a, st);
    if (a.K <= 16384) return run<TYPE, NORM, 16, 4>(a, st);
    return run<TYPE, NORM, 16, 0>(a, st);
}

}  // namespace

int i8_quantize_launch(const void *x, int type, long long ldx, const float *norm, float eps,
                       int8_t *q, long long ldq, float *s, int M, int K, int num_sms,
                       cudaStream_t stream) {
    const int esz = type == kI8F32 ? 4 : 2;
    const Args a{x, ldx, norm, eps, q, ldq, s, M, K,
                 (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * esz) % 16 == 0,
                 (reinterpret_cast<uintptr_t>(norm) & 15) == 0};
    const bool few = M < 2 * num_sms;
    switch (type) {
    case kI8F32: return norm ? pick<kI8F32, true>(a, few, stream) : pick<kI8F32, false>(a, few, stream);
    case kI8BF16:
        return norm ? pick<kI8BF16, true>(a, few, stream) : pick<kI8BF16, false>(a, few, stream);
    case kI8F16: return norm ? pick<kI8F16, true>(a, few, stream) : pick<kI8F16, false>(a, few, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace fb
