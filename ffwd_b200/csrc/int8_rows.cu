// Rows to 8-bit integers with one scale each (see int8.cuh), optionally after
// an RMSNorm.  Bound by memory: each row is read once into registers (rows of
// up to 16384 columns; longer ones are read twice) and written once at a byte
// per value.
//
// Rounding.  The code of a value is the nearest integer of v / s (s = amax / 127,
// both quotients in f64; ties to even).  In f32 the quotient is off by a few
// units in the last place, which matters only next to the border of two codes;
// there it is taken again in f64: about one value in 10^5 of f32 rows, and of
// bf16 rows one in 450, which lie on a border exactly.  The row's RMS cancels
// out of v / s, so with `norm` the codes depend on x * norm alone and only the
// scale carries the RMS.  Rows below 1e-30 (the largest value, or with `norm` the
// largest product or the mean square) are worked on in f64 throughout.
#include "int8.cuh"
#include "launch_util.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace fb {
namespace {

template <int TYPE>
__device__ __forceinline__ float load1(const void *x, size_t i) {
    if (TYPE == kI8F32) return static_cast<const float *>(x)[i];
    const uint16_t h = static_cast<const uint16_t *>(x)[i];
    if (TYPE == kI8BF16) return __uint_as_float((uint32_t)h << 16);
    return __half2float(__ushort_as_half(h));
}

// How a row's columns map to loads: by element (kScalar: any K and alignment);
// by four values (kFour: K and the addresses are multiples of four; columns
// past K repeat the row's first ones, which changes no maximum); or by four
// with every column inside (kFull: no bounds at all).
enum Cover { kScalar, kFour, kFull };

// Eight values of a row as loaded, columns [c, c + 4) and [c + 128, c + 132):
// a warp whose lanes are 4 columns apart reads 256 columns in whole lines, of
// the row and of f32 norm weights alike.  16-bit types stay packed: half the
// registers, so twice the rows in flight.
template <int TYPE, int COVER>
struct Raw {
    uint32_t w[TYPE == kI8F32 ? 8 : 4];

    __device__ __forceinline__ void load(const void *x, size_t off, int c, int K) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int ch = c + 128 * h;
            if (COVER == kFour) ch = ch < K ? ch : 0;
            if (TYPE == kI8F32) {
                const uint32_t *p = static_cast<const uint32_t *>(x) + off + ch;
                if (COVER != kScalar) {
                    const uint4 r = ld_global(reinterpret_cast<const uint4 *>(p));
                    w[4 * h] = r.x;
                    w[4 * h + 1] = r.y;
                    w[4 * h + 2] = r.z;
                    w[4 * h + 3] = r.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[4 * h + i] = ch + i < K ? p[i] : 0u;
                }
            } else {
                const uint16_t *p = static_cast<const uint16_t *>(x) + off + ch;
                if (COVER != kScalar) {
                    const uint2 r = ld_global(reinterpret_cast<const uint2 *>(p));
                    w[2 * h] = r.x;
                    w[2 * h + 1] = r.y;
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t lo = ch + 2 * i < K ? p[2 * i] : 0u;
                        const uint32_t hi = ch + 2 * i + 1 < K ? p[2 * i + 1] : 0u;
                        w[2 * h + i] = lo | hi << 16;
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (TYPE == kI8F32) {
                v[2 * i] = __uint_as_float(w[2 * i]);
                v[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
            } else if (TYPE == kI8BF16) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
};

template <int COVER>
__device__ __forceinline__ void load_norm(const float *w, int c, int K, float (&g)[8]) {
    Raw<kI8F32, COVER> r;
    r.load(w, 0, c, K);
    r.unpack(g);
}

// v / s in f64, correctly rounded, given rs = 1 / s to nearly f64's precision
// (the quotient's first estimate and one correction from its exact remainder).
__device__ __forceinline__ double quotient(double v, double s, double rs) {
    const double t = v * rs;
    return fma(fma(-t, s, v), rs, t);
}

// max(m, |a|, |b|), NaN if one is.
__device__ __forceinline__ float max_abs(float m, float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
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

__device__ __forceinline__ float pick8(const float (&v)[8], int j) {
    const float a = j & 1 ? v[1] : v[0], b = j & 1 ? v[3] : v[2];
    const float c = j & 1 ? v[5] : v[4], d = j & 1 ? v[7] : v[6];
    const float e = j & 2 ? b : a, f = j & 2 ? d : c;
    return j & 4 ? f : e;
}

// Codes of eight values (x, or x * g with a norm) of a row whose largest
// magnitude is amax + amax_lo, written at columns c and c + 128 on.  With SETTLE, values next to a border are settled; without, the result
// says whether there are any.
template <bool NORM, bool SETTLE, int COVER>
__device__ __forceinline__ bool put8(float (&x)[8], const float (&g)[8], float inv, float amax,
                                     float amax_lo, int8_t *q, int c, int K) {
    // How far the f32 quotient may be off: 127 x 2^-24 for the reciprocal's
    // rounding; with a norm as much again for the product's and for amax's.
    constexpr float kBand = NORM ? 2.6e-5f : 1e-5f;
    float code[8], d[8];
    float far = 0.0f;  // largest distance from a code
    const float2 inv2 = make_float2(inv, inv), up = make_float2(kRound, kRound),
                 minus = make_float2(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 t = make_float2(x[2 * i], x[2 * i + 1]);
        if (NORM) t = mul_f32x2(t, make_float2(g[2 * i], g[2 * i + 1]));
        const float2 f = fma_f32x2(t, inv2, up);
        const float2 r = fma_f32x2(t, inv2, fma_f32x2(f, minus, up));
        far = max_abs(far, r.x, r.y);
        code[2 * i] = f.x;
        code[2 * i + 1] = f.y;
        d[2 * i] = r.x;
        d[2 * i + 1] = r.y;
    }
    uint32_t w0 = low_bytes(code[0], code[1], code[2], code[3]);
    uint32_t w1 = low_bytes(code[4], code[5], code[6], code[7]);
    const bool any = far > 0.5f - kBand;
    if (SETTLE && any) {
        // In f64, one value after another (a rare path, kept small).  s = amax /
        // 127 likewise; 1 / s from inv in two Newton steps.
        const double am = (double)amax + (double)amax_lo;
        const double s = quotient(am, 127.0, 1.0 / 127.0);
        double rs = (double)inv;
        rs = fma(fma(-s, rs, 1.0), rs, rs);
        rs = fma(fma(-s, rs, 1.0), rs, rs);
        uint32_t near = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) near |= fabsf(d[i]) > 0.5f - kBand ? 1u << i : 0u;
#pragma unroll 1
        for (; near; near &= near - 1) {
            const int j = __ffs(near) - 1;
            double v = (double)pick8(x, j);
            if (NORM) v *= (double)pick8(g, j);
            const uint32_t byte = (uint32_t)__double2int_rn(quotient(v, s, rs)) & 0xFF;
            const int sh = 8 * (j & 3);
            const uint32_t w = ((j < 4 ? w0 : w1) & ~(0xFFu << sh)) | byte << sh;
            if (j < 4) w0 = w;
            else w1 = w;
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int ch = c + 128 * h;
        const uint32_t w = h ? w1 : w0;
        if (COVER != kScalar) {
            if (COVER == kFull || ch < K) *reinterpret_cast<uint32_t *>(q + ch) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (ch + i < K) q[ch + i] = (int8_t)(w >> (8 * i));
        }
    }
    return any;
}

// Zeros at columns c and c + 128 on.
template <int COVER>
__device__ __forceinline__ void zero8(int8_t *q, int c, int K) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int ch = c + 128 * h;
        if (COVER != kScalar) {
            if (COVER == kFull || ch < K) *reinterpret_cast<uint32_t *>(q + ch) = 0u;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (ch + i < K) q[ch + i] = 0;
        }
    }
}

// Blocks per SM that the registers allow: the row's values twice (this row's
// and the next one's, in flight).
constexpr int min_blocks(int type, bool norm, int w, int nv) {
    const int regs = 40 + nv * (type == kI8F32 ? 16 : 8) + (norm ? 8 : 0);
    const int n = 65536 / ((w == 1 ? 8 : w) * 32 * regs);
    return n < 1 ? 1 : n > 12 ? 12 : n;
}

// W warps per row, each thread holding NV groups of 8 columns (NV = 0: any
// width, the row read again in each pass).  A block of W (8 for W = 1) warps walks
// over rows, the next row's loads in flight while it works on one.
template <int TYPE, bool NORM, int COVER, int W, int NV>
__global__ void __launch_bounds__((W == 1 ? 8 : W) * 32, min_blocks(TYPE, NORM, W, NV))
    quantize_kernel(const void *x, long long ldx, const float *norm, float eps, int8_t *q,
                    long long ldq, float *s, int M, int K) {
    constexpr int NW = W == 1 ? 8 : W, R = NW / W;  // rows of a block at a time
    __shared__ uint32_t sh_max[NW];
    __shared__ float sh_sum[NW], sh_lo[NW];
    __shared__ double sh_max64[NORM ? NW : 1], sh_sum64[NORM ? NW : 1];
    griddep_wait();
    griddep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int wr = warp % W;  // warp of the row
    const int t = wr * 32 + lane;
    const int c0 = wr * 256 + lane * 4;  // first column of this thread's groups
    constexpr int NR = NV > 0 ? NV : 1;
    Raw<TYPE, COVER> next[NR];
    auto prefetch = [&](int row) {
        if (NV > 0 && row < M) {
#pragma unroll
            for (int k = 0; k < NR; ++k)
                next[k].load(x, (size_t)row * ldx, k * W * 256 + c0, K);
        }
    };
    const int stride = gridDim.x * R;
    prefetch(blockIdx.x * R + warp / W);
    // (the block's rounds are counted by its first row: all of its warps take part)
#pragma unroll 1
    for (int left = M - blockIdx.x * R; left > 0; left -= stride) {
        const int row = M - left + warp / W;
        const bool live = row < M;
        const size_t off = live ? (size_t)row * ldx : 0;
        Raw<TYPE, COVER> raw[NR];
#pragma unroll
        for (int k = 0; k < NR; ++k) raw[k] = next[k];
        if (left > stride) prefetch(row + stride);
        // Each of the passes over the row below: from registers, or loaded again.
        auto each = [&](auto f) {
            float v[8], g[8];
            if (NV > 0) {
                // (f32 rows: the next group's weights on their way while one is worked
                // on; rows of 16 bits have no registers for them, 8192 x 4096 f16 31
                // us without, 34 with spills)
                Raw<kI8F32, COVER> w;
                if (NORM && TYPE == kI8F32) w.load(norm, 0, c0, K);
#pragma unroll
                for (int k = 0; k < NR; ++k) {
                    const int c = k * W * 256 + c0;
                    raw[k].unpack(v);
                    if (NORM && TYPE != kI8F32) w.load(norm, 0, c, K);
                    if (NORM) w.unpack(g);
                    if (NORM && TYPE == kI8F32 && k + 1 < NR) w.load(norm, 0, c + W * 256, K);
                    f(v, g, c);
                }
            } else {
                for (int c = c0; c < K; c += W * 256) {
                    raw[0].load(x, off, c, K);
                    raw[0].unpack(v);
                    if (NORM) load_norm<COVER>(norm, c, K, g);
                    f(v, g, c);
                }
            }
        };
        float2 m2 = make_float2(0.0f, 0.0f), s2 = m2;
        if (live)
            each([&](const float(&a)[8], const float(&b)[8], int c) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 v = make_float2(a[2 * i], a[2 * i + 1]);
                    if (NORM) {
                        if (COVER != kFour || c + i / 2 * 128 < K) s2 = fma_f32x2(v, v, s2);
                        v = mul_f32x2(v, make_float2(b[2 * i], b[2 * i + 1]));
                    }
                    if (i & 1)
                        m2.x = max_abs(m2.x, v.x, v.y);
                    else
                        m2.y = max_abs(m2.y, v.x, v.y);
                }
            });
        const float mv = max_abs(0.0f, m2.x, m2.y);
        float ss = s2.x + s2.y;
        // Magnitudes compare as unsigned integers, NaN above infinity.
        const uint32_t mine = __float_as_uint(mv);
        uint32_t mx = __reduce_max_sync(0xffffffffu, mine);
        if (NORM) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
        if (W > 1) {
            __syncthreads();  // the last round's reads are done
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
        const bool finite = mx < 0x7F800000u && (!NORM || ss < INFINITY);
        // (a mean square below 1e-30: the squares may have left f32)
        const bool plain = live && finite && amax >= 1e-30f &&
                           (!NORM || fmaf(eps, (float)K, ss) >= 1e-30f * (float)K);
        int8_t *qr = q + (size_t)row * ldq;
        if (plain && t == 0)
            s[row] = NORM ? amax / 127.0f / sqrtf(ss / (float)K + eps) : amax / 127.0f;
        const float inv = 127.0f / amax;
        bool open = false;  // codes left to settle
        if (plain)
            each([&](float(&a)[8], const float(&b)[8], int c) {
                if (COVER == kFull || c < K) open |= put8<NORM, !NORM, COVER>(a, b, inv, amax, 0.0f, qr, c, K);
            });
        if (live && !plain) {
            // 127 / amax may pass f32 for rows so small, and their products with
            // the weights and their squares may be below it: a value at a time, in
            // f64 (W > 1: a row is all of the block's, so the block meets here).
            // Rows of zeros, or not finite, get zeros.
            double am = finite ? amax : 0.0f, rms = 1.0;
            bool some = finite;
            if (NORM && mx == 0) {  // zeros, or products below f32
                some = false;
                each([&](const float(&a)[8], const float(&)[8], int) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) some |= a[i] != 0.0f;
                });
                some = W == 1 ? __any_sync(0xffffffffu, some) : __syncthreads_or(some);
            }
            if (NORM && some) {
                double sq = 0.0;
                am = 0.0;
#pragma unroll 1
                for (int c = t; c < K; c += W * 32) {
                    const double v = (double)load1<TYPE>(x, off + c);
                    am = fmax(am, fabs(v * (double)norm[c]));
                    sq = fma(v, v, sq);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    am = fmax(am, __shfl_xor_sync(0xffffffffu, am, o));
                    sq += __shfl_xor_sync(0xffffffffu, sq, o);
                }
                if (W > 1) {
                    if (lane == 0) {
                        sh_max64[warp] = am;
                        sh_sum64[warp] = sq;
                    }
                    __syncthreads();
                    sq = 0.0;
#pragma unroll 1
                    for (int i = 0; i < W; ++i) {
                        am = fmax(am, sh_max64[i]);
                        sq += sh_sum64[i];
                    }
                }
                rms = sqrt(sq / (double)K + (double)eps);
            }
            const double sc = am / 127.0;
            if (t == 0) s[row] = finite ? (float)(sc / rms) : __uint_as_float(0x7FC00000u);
#pragma unroll 1
            for (int c = t; am > 0.0 && c < K; c += W * 32) {
                double v = (double)load1<TYPE>(x, off + c);
                if (NORM) v *= (double)norm[c];
                qr[c] = (int8_t)(int)rint(v / sc);
            }
            if (!(am > 0.0))
#pragma unroll 1
                for (int c = c0; c < K; c += W * 256) zero8<COVER>(qr, c, K);
        }
        if (NORM) {
            // Settling takes the largest product in full: among the values whose
            // rounded product is the maximum, the largest residue (rounding
            // keeps the order).  Few rows need it.
            if (!(W == 1 ? __any_sync(0xffffffffu, open) : __syncthreads_or(open))) continue;
            float lo = -INFINITY;
            if (plain && mine == mx)
                each([&](const float(&a)[8], const float(&b)[8], int) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float p = a[i] * b[i];
                        if (fabsf(p) == amax) {
                            const float e = fmaf(a[i], b[i], -p);
                            lo = fmaxf(lo, p < 0.0f ? -e : e);
                        }
                    }
                });
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
            if (open)
                each([&](float(&a)[8], const float(&b)[8], int c) {
                    if (COVER == kFull || c < K) put8<NORM, true, COVER>(a, b, inv, amax, lo, qr, c, K);
                });
        }
    }
}

// LayerNorm of f32 rows in place, their codes written beside them: a warp per
// row (at most NV x 256 columns), the row in registers, the next one's loads in
// flight.  Replaces a LayerNorm and a quantisation (15 bytes a value with the
// 16-bit copy between them) by 9 bytes a value.
template <int COVER, int NV>
__global__ void __launch_bounds__(256, 2)
    layernorm_quantize_kernel(float *x, const float *gamma, const float *beta, float eps,
                              int8_t *q, float *s, int M, int K) {
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31;
    const int stride = gridDim.x * 8;
    int row = blockIdx.x * 8 + (threadIdx.x >> 5);
    Raw<kI8F32, COVER> next[NV];
    auto prefetch = [&](int r) {
#pragma unroll
        for (int k = 0; k < NV; ++k) next[k].load(x, (size_t)r * K, k * 256 + lane * 4, K);
    };
    auto sum = [&](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    if (row < M) prefetch(row);
#pragma unroll 1
    for (; row < M; row += stride) {
        float v[NV][8];
#pragma unroll
        for (int k = 0; k < NV; ++k) next[k].unpack(v[k]);
        if (M - row > stride) prefetch(row + stride);
        // (k, i) -> whether the value's column is inside the row
        auto in = [&](int k, int i) {
            return COVER == kFull || k * 256 + lane * 4 + i / 4 * 128 < K;
        };
        float acc = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (in(k, i)) acc += v[k][i];
        const float mean = sum(acc) / (float)K;
        acc = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[k][i] -= mean;
                if (in(k, i)) acc = fmaf(v[k][i], v[k][i], acc);
            }
        const float inv_std = 1.0f / sqrtf(sum(acc) / (float)K + eps);
        float mv = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = k * 256 + lane * 4;
            float g[8], b[8];
            load_norm<COVER>(gamma, c, K, g);
            load_norm<COVER>(beta, c, K, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = fmaf(g[i] * v[k][i], inv_std, b[i]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (in(k, 4 * h))
                    *reinterpret_cast<float4 *>(x + (size_t)row * K + c + 128 * h) = make_float4(
                        v[k][4 * h], v[k][4 * h + 1], v[k][4 * h + 2], v[k][4 * h + 3]);
            // (columns past the row repeat valid ones, through other weights' places)
#pragma unroll
            for (int i = 0; i < 8; i += 2)
                if (in(k, i)) mv = max_abs(mv, v[k][i], v[k][i + 1]);
        }
        const uint32_t mx = __reduce_max_sync(0xffffffffu, __float_as_uint(mv));
        const float amax = __uint_as_float(mx);
        const bool finite = mx < 0x7F800000u;
        if (lane == 0) s[row] = finite ? amax / 127.0f : __uint_as_float(0x7FC00000u);
        const float inv = finite && amax >= 1e-30f ? 127.0f / amax : 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = k * 256 + lane * 4;
            if (inv == 0.0f) {  // zeros, or not finite: no codes
#pragma unroll
                for (int i = 0; i < 8; ++i) v[k][i] = 0.0f;
            }
            if (COVER == kFull || c < K)
                put8<false, true, COVER>(v[k], v[k], inv, inv == 0.0f ? 1.0f : amax, 0.0f,
                                         q + (size_t)row * K, c, K);
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
    int M, K, num_sms;
};

template <int TYPE, bool NORM, int COVER, int W, int NV>
cudaError_t run(const Args &a, cudaStream_t st) {
    constexpr int NW = W == 1 ? 8 : W, R = NW / W;
    const int grid = std::min((a.M + R - 1) / R, a.num_sms * min_blocks(TYPE, NORM, W, NV));
    return launch_k(quantize_kernel<TYPE, NORM, COVER, W, NV>, dim3(grid), dim3(NW * 32), 0, st,
                    a.x, a.ldx, a.norm, a.eps, a.q, a.ldq, a.s, a.M, a.K);
}

// W warps a row, NV groups a thread where they cover the row exactly.
template <int TYPE, bool NORM, int W>
cudaError_t full(const Args &a, cudaStream_t st) {
    switch (a.K / (W * 256)) {
    case 1: return run<TYPE, NORM, kFull, W, 1>(a, st);
    case 2: return run<TYPE, NORM, kFull, W, 2>(a, st);
    case 3: return run<TYPE, NORM, kFull, W, 3>(a, st);
    }
    return run<TYPE, NORM, kFull, W, 4>(a, st);
}

// Many rows: as few warps per row as hold it (a warp's own reductions, no
// block barrier), without bounds where its width is a whole number of groups
// (32768 x 1024 f32 with norm: 34 us with them).  Few rows (under two per SM):
// more warps per row, so that a row's loads are all in flight at once.
// Columns or addresses that are no multiple of four values: by element, the row
// read again in each pass.
template <int TYPE, bool NORM>
cudaError_t pick(const Args &a, bool vec, cudaStream_t st) {
    const bool few = a.M < 2 * a.num_sms;
    if (!vec) {
        return a.K <= 1024 && !few ? run<TYPE, NORM, kScalar, 1, 0>(a, st)
                                   : run<TYPE, NORM, kScalar, 16, 0>(a, st);
    }
    if (few) {
        if (a.K <= 1024) return run<TYPE, NORM, kFour, 4, 1>(a, st);
        if (a.K <= 4096) return run<TYPE, NORM, kFour, 16, 1>(a, st);
    } else {
        if (a.K <= 1024)
            return a.K % 256 == 0   ? full<TYPE, NORM, 1>(a, st)
                   : a.K <= 512 ? run<TYPE, NORM, kFour, 1, 2>(a, st)
                                : run<TYPE, NORM, kFour, 1, 4>(a, st);
        if (a.K <= 4096)
            return a.K % 1024 == 0 ? full<TYPE, NORM, 4>(a, st)
                                   : run<TYPE, NORM, kFour, 4, 4>(a, st);
        if (a.K <= 16384 && a.K % 4096 == 0) return full<TYPE, NORM, 16>(a, st);
    }
    if (a.K <= 16384) return run<TYPE, NORM, kFour, 16, 4>(a, st);
    return run<TYPE, NORM, kFour, 16, 0>(a, st);
}

}  // namespace

int i8_quantize_launch(const void *x, int type, long long ldx, const float *norm, float eps,
                       int8_t *q, long long ldq, float *s, int M, int K, int num_sms,
                       cudaStream_t stream) {
    const uintptr_t four = type == kI8F32 ? 16 : 8;  // bytes of four values
    const bool vec = reinterpret_cast<uintptr_t>(x) % four == 0 && ldx % 4 == 0 && K % 4 == 0 &&
                     reinterpret_cast<uintptr_t>(norm) % 16 == 0;
    const Args a{x, ldx, norm, eps, q, ldq, s, M, K, num_sms};
    switch (type) {
    case kI8F32: return norm ? pick<kI8F32, true>(a, vec, stream) : pick<kI8F32, false>(a, vec, stream);
    case kI8BF16:
        return norm ? pick<kI8BF16, true>(a, vec, stream) : pick<kI8BF16, false>(a, vec, stream);
    case kI8F16: return norm ? pick<kI8F16, true>(a, vec, stream) : pick<kI8F16, false>(a, vec, stream);
    }
    return cudaErrorInvalidValue;
}

bool i8_layernorm_quantize_fits(int K) { return K <= 1024 && K % 16 == 0; }

int i8_layernorm_quantize_launch(float *x, const float *gamma, const float *beta, float eps,
                                 int8_t *q, float *s, int M, int K, int num_sms,
                                 cudaStream_t stream) {
    const int grid = std::min((M + 7) / 8, num_sms * 2);
    auto go = [&](auto kern) {
        return launch_k(kern, dim3(grid), dim3(256), 0, stream, x, gamma, beta, eps, q, s, M, K);
    };
    switch (K) {
    case 256: return go(layernorm_quantize_kernel<kFull, 1>);
    case 512: return go(layernorm_quantize_kernel<kFull, 2>);
    case 768: return go(layernorm_quantize_kernel<kFull, 3>);
    case 1024: return go(layernorm_quantize_kernel<kFull, 4>);
    }
    return K <= 512 ? go(layernorm_quantize_kernel<kFour, 2>) : go(layernorm_quantize_kernel<kFour, 4>);
}

}  // namespace fb
