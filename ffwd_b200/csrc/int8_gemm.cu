// Two-SM tcgen05 kernel of the 8-bit integer projections (kind::i8, s8 x s8
// with 32-bit integer sums).
//
// A cluster of two CTAs computes a 256 x BN tile: each CTA holds 128 rows of
// the quantised rows and half of the tile's weight rows in shared memory (128
// bytes of K per stage row, 128-byte swizzle), the leader issues
// tcgen05.mma.cta_group::2 (M = 256, N = BN, K = 32 bytes) and each CTA keeps
// its 128 output rows in TMEM, in two accumulators, so a tile's epilogue runs
// under the next tile's products.  In the gated form the leader's half of the
// weight rows are the gate's and its peer's the up projection's, so matching
// columns meet in one accumulator.  Roles per CTA (320 threads): warp 0 TMA
// producer, warp 1 TMEM allocation and (leader) MMA issue, warps 2-9 epilogue
// in two warpgroups that split the columns.  No TMA load uses multicast.
#include "gemm_epi.cuh"
#include "host_util.h"
#include "int8.cuh"
#include "int8_epi.cuh"
#include "launch_util.cuh"
#include "ptx.cuh"

#include <algorithm>

namespace fb {
namespace {

constexpr int BM = 128;       // rows per CTA
constexpr int BK = 128;       // bytes of K per stage
constexpr int kGroups = 2;    // epilogue warpgroups
constexpr int kThreads = 64 + 128 * kGroups;
constexpr int A_BYTES = BM * BK;
constexpr int CHUNK = 8192;   // 128 rows x 64 bytes of output
constexpr uint32_t kPeerMask = 0xFEFFFFFFu;  // clears the CTA-rank bit: leader's copy

template <int BN>
struct Cfg {
    static constexpr int B_BYTES = (BN / 2) * BK;  // this CTA's half of the weight rows
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = BN == 256 ? 5 : BN == 128 ? 7 : 8;
    static constexpr int OFF_STAGING = STAGES * STAGE;
    static constexpr int OFF_COLS = OFF_STAGING + kGroups * 2 * CHUNK;
    // Per warpgroup: the tile's scales and biases.
    static constexpr int SMEM = OFF_COLS + kGroups * 2 * BN * 4 + 1024;
    static constexpr int TMEM_COLS = 2 * BN;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                     : "memory");
}

// Tile load into this CTA's shared memory, bytes counted on the leader's barrier.
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *m, uint32_t bar_leader,
                                              int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_leader), "r"(x), "r"(y)
        : "memory");
}

// D[tmem, s32] (+)= A * B^T, 8-bit integers.
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum)
        : "memory");
}

// Instruction descriptor, kind::i8: s32 accumulate, both operands signed, K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

// Arrive on the barrier at this offset in both CTAs once the issued MMAs complete.
__device__ __forceinline__ void umma_commit_pair(uint64_t *bar) {
    const uint16_t mask = 0x3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(smem_u32(bar)),
        "h"(mask)
        : "memory");
}

__device__ __forceinline__ void arrive_leader(uint64_t *bar) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(smem_u32(bar)));
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote)
                 : "memory");
}

// Output of one warpgroup: 64-byte row segments (32 16-bit or 16 f32 columns)
// staged in shared memory with the 64-byte swizzle, then one TMA store (or
// f32 reduce-add) per chunk; where the output's base or row stride is not a
// multiple of 16 bytes, the chunk's elements are written by the warps, a row
// segment per (half) warp.  Rows past M and columns past N are left alone.
struct Sink {
    const I8Params &p;
    const CUtensorMap *map;
    uint8_t *stage;  // two chunks
    int r, y0, g;
    bool elected, tma;
    int k = 0;

    __device__ __forceinline__ uint8_t *acquire() {
        uint8_t *buf = stage + (k & 1) * CHUNK;
        if (elected && tma) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        named_bar(1 + g, 128);
        return buf;
    }
    __device__ __forceinline__ void publish(uint8_t *buf, int col) {
        if (tma) fence_proxy_async_smem();
        named_bar(1 + g, 128);
        if (tma) {
            if (elected) {
                if (p.accumulate)
                    asm volatile(
                        "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group"
                        " [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
                        "r"(smem_u32(buf)), "r"(col), "r"(y0)
                        : "memory");
                else
                    asm volatile(
                        "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group"
                        " [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
                        "r"(smem_u32(buf)), "r"(col), "r"(y0)
                        : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        } else {
            const int lane = r & 31, w = r >> 5;
            const bool f32 = p.type == kI8F32;
            const int width = f32 ? 16 : 32;
            const int c = lane & (width - 1);
            const int byte = f32 ? c * 4 : c * 2;
            if (col + c < p.N) {
                const int rows = min(BM, p.M - y0);
                for (int i = f32 ? 2 * w + (lane >> 4) : w; i < rows; i += f32 ? 8 : 4) {
                    const uint8_t *src =
                        buf + i * 64 + (((byte >> 4) ^ ((i >> 1) & 3)) << 4) + (byte & 15);
                    const size_t off = (size_t)(y0 + i) * p.ldy + col + c;
                    if (f32) {
                        float *o = static_cast<float *>(p.y) + off;
                        const float v = *reinterpret_cast<const float *>(src);
                        *o = p.accumulate ? *o + v : v;
                    } else {
                        static_cast<uint16_t *>(p.y)[off] = *reinterpret_cast<const uint16_t *>(src);
                    }
                }
            }
        }
        ++k;
    }
    // 32 columns [col, col + 32) of this thread's row.
    __device__ __forceinline__ void put(const float (&v)[32], int col) {
        if (p.type == kI8F32) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (col + 16 * h >= p.N) break;
                uint8_t *buf = acquire();
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<float4 *>(buf + r * 64 + ((c ^ ((r >> 1) & 3)) * 16)) =
                        make_float4(v[16 * h + 4 * c], v[16 * h + 4 * c + 1],
                                    v[16 * h + 4 * c + 2], v[16 * h + 4 * c + 3]);
                publish(buf, col + 16 * h);
            }
            return;
        }
        uint8_t *buf = acquire();
        const bool f16 = p.type == kI8F16;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4 *>(buf + r * 64 + ((c ^ ((r >> 1) & 3)) * 16)) =
                make_uint4(pack16x2(v[8 * c], v[8 * c + 1], f16),
                           pack16x2(v[8 * c + 2], v[8 * c + 3], f16),
                           pack16x2(v[8 * c + 4], v[8 * c + 5], f16),
                           pack16x2(v[8 * c + 6], v[8 * c + 7], f16));
        publish(buf, col);
    }
    __device__ __forceinline__ void finish() {
        if (elected && tma) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
};

// 32 accumulators scaled: v = acc * s * t + b.
__device__ __forceinline__ void scale32(float (&v)[32], float s, const float *t, const float *b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 tv = reinterpret_cast<const float4 *>(t)[i];
        const float4 bv = reinterpret_cast<const float4 *>(b)[i];
        const float tt[4] = {tv.x, tv.y, tv.z, tv.w}, bb[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
            v[4 * i + u] = fmaf((float)__float_as_int(v[4 * i + u]) * s, tt[u], bb[u]);
    }
}

__device__ __forceinline__ void act32(float (&v)[32], int act, bool f32) {
    if (act == kI8None) return;
    if (act == kI8Silu && !f32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = epi::silu_fast(v[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = i8::act_full(v[i], act);
}

// One 128-row x BN accumulator.  cols: this warpgroup's scales [BN] then biases [BN].
template <int BN, int EPI, int HD>
__device__ __forceinline__ void epilogue(const I8Params &p, uint32_t tbase, int grow, float s,
                                         int nb, int g, const float *cols, Sink &sink) {
    const bool f32 = p.type == kI8F32;
    if constexpr (EPI == kI8Store) {
#pragma unroll 1
        for (int c = g; c < BN / 32; c += kGroups) {
            const int col = nb * BN + c * 32;
            if (col >= p.N) break;
            float v[32];
            tmem_ld32(tbase + c * 32, v);
            tmem_wait_ld();
            scale32(v, s, cols + c * 32, cols + BN + c * 32);
            act32(v, p.act, f32);
            sink.put(v, col);
        }
    } else if constexpr (EPI == kI8Gated) {
#pragma unroll 1
        for (int c = g; c < BN / 64; c += kGroups) {
            const int col = nb * (BN / 2) + c * 32;
            if (col >= p.N) break;
            float a[32], u[32];
            tmem_ld32(tbase + c * 32, a);
            tmem_ld32(tbase + BN / 2 + c * 32, u);
            tmem_wait_ld();
            scale32(a, s, cols + c * 32, cols + BN + c * 32);
            scale32(u, s, cols + BN / 2 + c * 32, cols + BN + BN / 2 + c * 32);
            act32(a, p.act, f32);
#pragma unroll
            for (int i = 0; i < 32; ++i) a[i] *= u[i];
            sink.put(a, col);
        }
    } else {
        constexpr int HALF = HD / 2;
#pragma unroll 1
        for (int h0 = g * HD; h0 < BN; h0 += kGroups * HD) {
            const int col0 = nb * BN + h0;
            if (col0 >= p.N) break;
            const int head = col0 / HD;
            const bool is_q = head < p.n_q_heads;
            const bool rot = head < p.n_q_heads + p.n_kv_heads;
            float v[HD / 32][32];
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) tmem_ld32(tbase + h0 + c * 32, v[c]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < HD / 32; ++c)
                scale32(v[c], s, cols + h0 + c * 32, cols + BN + h0 + c * 32);
            if (rot) {
                const float *nw = is_q ? p.q_norm : p.k_norm;
                const int ps = grow < p.M ? __ldg(p.pos + grow) : 0;
                const bool bad = ps < 0 || ps >= p.n_pos;
                if (bad) set_error(p.err, kErrBadPosition);
                float inv = bad ? i8::nan_f() : 1.0f;
                if (nw) {
                    float ss = 0.0f;
#pragma unroll
                    for (int c = 0; c < HD / 32; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) ss = fmaf(v[c][i], v[c][i], ss);
                    inv *= 1.0f / sqrtf(ss / (float)HD + p.eps);
                }
                const float4 *cs =
                    reinterpret_cast<const float4 *>(p.cos + (size_t)(bad ? 0 : ps) * HALF);
                const float4 *sn =
                    reinterpret_cast<const float4 *>(p.sin + (size_t)(bad ? 0 : ps) * HALF);
#pragma unroll
                for (int i = 0; i < HALF / 4; ++i) {
                    const float4 cv = __ldg(cs + i), sv = __ldg(sn + i);
                    float4 w1 = make_float4(1.0f, 1.0f, 1.0f, 1.0f), w2 = w1;
                    if (nw) {
                        w1 = __ldg(reinterpret_cast<const float4 *>(nw) + i);
                        w2 = __ldg(reinterpret_cast<const float4 *>(nw + HALF) + i);
                    }
                    const float cc[4] = {cv.x, cv.y, cv.z, cv.w}, sc[4] = {sv.x, sv.y, sv.z, sv.w};
                    const float wa[4] = {w1.x, w1.y, w1.z, w1.w}, wb[4] = {w2.x, w2.y, w2.z, w2.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        constexpr int H32 = HALF / 32;
                        const int e = 4 * i + u;
                        float &a = v[e / 32][e % 32], &b = v[H32 + e / 32][e % 32];
                        const float x1 = a * inv * wa[u], x2 = b * inv * wb[u];
                        a = x1 * cc[u] - x2 * sc[u];
                        b = x2 * cc[u] + x1 * sc[u];
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) sink.put(v[c], col0 + c * 32);
        }
    }
}

template <int BN, int EPI, int HD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    i8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmB2,
                   const __grid_constant__ CUtensorMap tmOut, const I8Params p, const int tma_out) {
    extern __shared__ uint8_t smem_raw[];
    using CF = Cfg<BN>;
    constexpr int STAGES = CF::STAGES;
    __shared__ __align__(8) uint64_t full_bar[STAGES];
    __shared__ __align__(8) uint64_t empty_bar[STAGES];
    __shared__ __align__(8) uint64_t tfull_bar[2];
    __shared__ __align__(8) uint64_t tempty_bar[2];
    __shared__ __align__(8) uint64_t drain_bar;
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_sh;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));

    constexpr int TN = EPI == kI8Gated ? BN / 2 : BN;  // output columns per tile
    const int m_blocks = (p.M + 2 * BM - 1) / (2 * BM);
    const int n_blocks = (p.N + TN - 1) / TN;
    const int num_tiles = m_blocks * n_blocks;
    const int k_blocks = (p.K + BK - 1) / BK;
    const int pair = blockIdx.x >> 1;
    const int n_pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull_bar[a], 1);
            mbar_init(&tempty_bar[a], 2 * 4 * kGroups);
        }
        mbar_init(&drain_bar, 1);
        abort_sh = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        if (EPI == kI8Gated) tma_prefetch_desc(&tmB2);
        if (tma_out) tma_prefetch_desc(&tmOut);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_base_sh)),
                     "r"(CF::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers initialised before any remote use
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_sh;
    griddep_wait();
    griddep_launch();

    if (warp == 0) {
        if (lane == 0) {
            // ---------------------------------------------------------- producer
            const CUtensorMap *mb_map = EPI == kI8Gated && !leader ? &tmB2 : &tmB;
            int it = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < num_tiles; tile += n_pairs) {
                const int mb = tile / n_blocks, nb = tile % n_blocks;
                const int brow = EPI == kI8Gated ? nb * TN : nb * BN + (int)rank * (BN / 2);
                for (int kb = 0; kb < k_blocks; ++kb) {
                    const int s = it % STAGES;
                    const uint32_t ph = (it / STAGES) & 1;
                    if (!mbar_wait(&empty_bar[s], ph ^ 1, p.err, &abort_sh)) {
                        ok = false;
                        break;
                    }
                    uint8_t *st = smem + s * CF::STAGE;
                    if (leader) mbar_arrive_expect_tx(&full_bar[s], 2 * CF::STAGE);
                    const uint32_t bar = smem_u32(&full_bar[s]) & kPeerMask;
                    tma_load_pair(st, &tmA, bar, kb * BK, mb * 2 * BM + rank * BM);
                    tma_load_pair(st + A_BYTES, mb_map, bar, kb * BK, brow);
                    ++it;
                }
            }
            if (!ok && leader) {
                for (int j = it - STAGES < 0 ? 0 : it - STAGES; j < it; ++j)
                    mbar_wait(&full_bar[j % STAGES], (j / STAGES) & 1, nullptr, nullptr);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (leader && lane == 0) {
            // ---------------------------------------------------------- MMA issuer
            constexpr uint32_t IDESC = idesc_i8(2 * BM, BN);
            int it = 0, lt = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < num_tiles; tile += n_pairs, ++lt) {
                const int a = lt & 1;
                const uint32_t aph = (lt >> 1) & 1;
                if (!mbar_wait(&tempty_bar[a], aph ^ 1, p.err, &abort_sh)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem_base + a * BN;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    const int s = it % STAGES;
                    const uint32_t ph = (it / STAGES) & 1;
                    if (!mbar_wait(&full_bar[s], ph, p.err, &abort_sh)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + s * CF::STAGE);
                    const uint32_t sb = sa + A_BYTES;
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk)
                        umma_i8_pair(d, smem_desc(sa + kk * 32, 16, 1024, kLayoutSW128),
                                     smem_desc(sb + kk * 32, 16, 1024, kLayoutSW128), IDESC,
                                     (kb | kk) != 0);
                    umma_commit_pair(&empty_bar[s]);
                    ++it;
                }
                if (!ok) break;
                umma_commit_pair(&tfull_bar[a]);
            }
            if (!ok) {
                asm volatile(
                    "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                        smem_u32(&drain_bar))
                    : "memory");
                mbar_wait(&drain_bar, 0, nullptr, nullptr);
            }
        }
        __syncwarp();
    } else {
        // -------------------------------------------------------------- epilogue
        const int q = warp & 3;
        const int g = (warp - 2) >> 2;
        const int row = q * 32 + lane;
        const int gt = (warp - 2 - 4 * g) * 32 + lane;  // thread of the warpgroup
        float *cols = reinterpret_cast<float *>(smem + CF::OFF_COLS) + g * 2 * BN;
        Sink sink{p, &tmOut, smem + CF::OFF_STAGING + g * 2 * CHUNK, row, 0, g, gt == 0,
                  tma_out != 0};
        int lt = 0;
        for (int tile = pair; tile < num_tiles; tile += n_pairs, ++lt) {
            const int a = lt & 1;
            const uint32_t aph = (lt >> 1) & 1;
            const int mb = tile / n_blocks, nb = tile % n_blocks;
            const int y0 = mb * 2 * BM + (int)rank * BM;
            const int grow = y0 + row;
            // The tile's scales and biases, fetched while its products run.  The
            // barrier ahead of the writes is past every read of the last tile's.
            const float s = grow < p.M ? __ldg(p.xs + grow) : 0.0f;
            named_bar(1 + g, 128);
            for (int c = gt; c < BN; c += 128) {
                const bool second = EPI == kI8Gated && c >= TN;
                const int col = nb * TN + (second ? c - TN : c);
                const float *t = second ? p.ws2 : p.ws, *b = second ? p.bias2 : p.bias;
                cols[c] = col < p.N ? __ldg(t + col) : 0.0f;
                cols[BN + c] = b && col < p.N ? __ldg(b + col) : 0.0f;
            }
            // One verdict for the warpgroup: its barriers below need all of it.
            if (!named_bar_and(1 + g, 128, mbar_wait(&tfull_bar[a], aph, p.err, &abort_sh))) break;
            tc_fence_after();
            const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + a * BN;
            sink.y0 = y0;
            if (y0 < p.M) epilogue<BN, EPI, HD>(p, tbase, grow, s, nb, g, cols, sink);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_leader(&tempty_bar[a]);
        }
        sink.finish();
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while its peer may still touch its barriers or smem
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                     "r"(CF::TMEM_COLS)
                     : "memory");
    }
}

template <int BN, int EPI, int HD>
int launch(const I8Params &p, int num_sms, cudaStream_t stream) {
    CUtensorMap ma, mb, mb2, mo;
    constexpr CUtensorMapDataType U8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    constexpr CUtensorMapSwizzle SW = CU_TENSOR_MAP_SWIZZLE_128B;
    if (make_map_ld(&ma, p.x, p.M, p.K, p.ldx, BM, BK, SW, U8, 1) ||
        make_map_ld(&mb, p.w, p.N, p.K, p.ldw, BN / 2, BK, SW, U8, 1))
        return -1;
    mb2 = mb;
    if (EPI == kI8Gated && make_map_ld(&mb2, p.w2, p.N, p.K, p.ldw2, BN / 2, BK, SW, U8, 1))
        return -1;
    const int esz = p.type == kI8F32 ? 4 : 2;
    const bool tma = (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && (p.ldy * esz) % 16 == 0;
    mo = ma;
    if (tma && make_map_ld(&mo, p.y, p.M, p.N, p.ldy, 128, 64 / esz, CU_TENSOR_MAP_SWIZZLE_64B,
                           p.type == kI8F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                           : p.type == kI8BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           esz))
        return -1;
    CK((set_smem_once<i8_gemm_kernel<BN, EPI, HD>>(Cfg<BN>::SMEM)));
    constexpr int TN = EPI == kI8Gated ? BN / 2 : BN;
    const long long tiles = (long long)((p.M + 2 * BM - 1) / (2 * BM)) * ((p.N + TN - 1) / TN);
    const int grid = (int)std::min<long long>(2 * tiles, num_sms & ~1);
    LAUNCH(launch_k(i8_gemm_kernel<BN, EPI, HD>, dim3(grid), dim3(kThreads), Cfg<BN>::SMEM, stream,
                    ma, mb, mb2, mo, p, tma ? 1 : 0));
    return 0;
}

// Tile width: waves of tiles over the SM pairs times the cost of a tile (its
// columns, plus a part that does not shrink with them: the 256 rows' loads
// and the pipeline's start).
int pick_bn(int epi, const I8Params &p, int num_sms) {
    const int pairs = std::max(1, num_sms / 2);
    const long long mb = (p.M + 2 * BM - 1) / (2 * BM);
    const long long cols = epi == kI8Gated ? 2ll * p.N : p.N;
    int best = 256;
    long long best_cost = -1;
    for (int bn : {256, 128, 64}) {
        if (epi == kI8Heads && bn < 128) break;
        const long long tiles = mb * ((cols + bn - 1) / bn);
        const long long cost = (tiles + pairs - 1) / pairs * (bn + 64);
        if (best_cost < 0 || cost < best_cost) {
            best = bn;
            best_cost = cost;
        }
    }
    return best;
}

template <int EPI, int HD>
int launch_bn(int bn, const I8Params &p, int num_sms, cudaStream_t stream) {
    if (bn == 256) return launch<256, EPI, HD>(p, num_sms, stream);
    if (bn == 128) return launch<128, EPI, HD>(p, num_sms, stream);
    if constexpr (EPI != kI8Heads) return launch<64, EPI, HD>(p, num_sms, stream);
    return -1;
}

}  // namespace

int i8_gemm_run(int epi, const I8Params &p, int num_sms, cudaStream_t stream) {
    const long long tiles = ((long long)p.M + 255) / 256 * (((long long)p.N + 31) / 32);
    if (tiles > INT32_MAX) {
        fail("8-bit product too large: %d x %d", p.M, p.N);
        return -1;
    }
    const int bn = pick_bn(epi, p, num_sms);
    switch (epi) {
    case kI8Store: return launch_bn<kI8Store, 0>(bn, p, num_sms, stream);
    case kI8Gated: return launch_bn<kI8Gated, 0>(bn, p, num_sms, stream);
    case kI8Heads:
        return p.head_dim == 128 ? launch_bn<kI8Heads, 128>(bn, p, num_sms, stream)
                                 : launch_bn<kI8Heads, 64>(bn, p, num_sms, stream);
    }
    return -1;
}

}  // namespace fb
