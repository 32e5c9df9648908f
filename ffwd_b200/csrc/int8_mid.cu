// 8-bit integer projections of a few tens of rows (see int8.cuh): latency and
// the weights' bytes bound them, not the products.  The operands change
// places, tcgen05.mma kind::i8 with 128 weight rows as M and T <= 128 quantised
// rows as N, so a weight byte costs T / 256 of the tensor work that the 256-row
// tiles of int8_gemm.cu spend on it; and where there are fewer 128-channel
// tiles than SMs, a cluster of S CTAs splits K: their integer sums meet in
// distributed shared memory, each CTA finishing T / S of the rows (exact, so
// the split changes no bit).  An accumulator column is a row of the result: a
// thread holds one channel (its scale and bias in registers), a warp stores 32
// neighbouring channels.
//
// Measured (weights in L2): 64 rows of 4096 x 12288 12 us, where the 256-row
// tiles take 28; of 1024 x 2048 6.1 us; of gate and up of 12288 x 4096 24 us
// (100 MB of weights: 15.6 us at the HBM rate).
//
// One tile per CTA.  Warp 0 TMA producer, warp 1 TMEM allocation and MMA issue,
// warps 2-9 the epilogue: two warpgroups that take turns at 8 rows.
#include "host_util.h"
#include "int8.cuh"
#include "int8_epi.cuh"
#include "launch_util.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <atomic>

namespace fb {
namespace {

constexpr int BK = 128;   // bytes of K per stage
constexpr int BC = 128;   // channels per tile
constexpr int kThreads = 64 + 256;
constexpr int kRows = 8;  // rows an epilogue warpgroup works on at once

template <int EPI, int T>
struct Cfg {
    static constexpr int MATS = EPI == kI8Gated ? 2 : 1;
    static constexpr int W_BYTES = BC * BK;
    static constexpr int STAGE = MATS * W_BYTES + T * BK;
    static constexpr int STAGES = 196608 / STAGE > 8 ? 8 : 196608 / STAGE;
    static constexpr int SMEM = STAGES * STAGE + 1024;
    static constexpr int TMEM_COLS = MATS * T < 32 ? 32 : MATS * T;
    // After the products the stages hold the sums [MATS][T][BC] and, in the head
    // form, values [T][BC] and partial sums of squares [T][4].
    static constexpr int OFF_VALUES = MATS * T * BC * 4;
    static_assert(OFF_VALUES + (EPI == kI8Heads ? T * (BC + 4) * 4 : 0) <= STAGES * STAGE,
                  "the sums fit the stages");
    static_assert(2 * SMEM > 227 * 1024, "one CTA to an SM (resident_clusters)");
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

// The int at this shared-memory address in CTA `rank` of the cluster.
__device__ __forceinline__ int load_peer(uint32_t addr, uint32_t rank) {
    int v;
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\t"
        "ld.shared::cluster.s32 %0, [a];\n\t}"
        : "=r"(v)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}

// (The operands' descriptors share their upper word.)
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi,
                                        uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accum)
        : "memory");
}

// kind::i8: s32 accumulate, both operands signed, K-major.
constexpr uint32_t idesc_i8(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

template <int EPI, int T, int HD>
__global__ void __launch_bounds__(kThreads)
    i8_mid_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmW2,
                  const __grid_constant__ CUtensorMap tmX, const I8Params p, const int split) {
    extern __shared__ uint8_t smem_raw[];
    using CF = Cfg<EPI, T>;
    constexpr int STAGES = CF::STAGES;
    __shared__ __align__(8) uint64_t full_bar[STAGES];
    __shared__ __align__(8) uint64_t empty_bar[STAGES];
    __shared__ __align__(8) uint64_t done_bar;
    __shared__ uint32_t tmem_base_sh;
    __shared__ int abort_sh;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int rank = split > 1 ? (int)cluster_rank() : 0;
    const int c0 = blockIdx.x / split * BC;  // first channel
    const int row0 = blockIdx.y * T;         // first row
    const int k_blocks = (p.K + BK - 1) / BK;
    const int kb0 = k_blocks * rank / split, kb1 = k_blocks * (rank + 1) / split;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&done_bar, 1);
        abort_sh = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmW);
        if (EPI == kI8Gated) tma_prefetch_desc(&tmW2);
        tma_prefetch_desc(&tmX);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_sh, CF::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_sh;
    // The first weights on their way to L2 while the stream's previous kernel
    // (as a rule the one that quantises the rows) still runs.
    if (threadIdx.x == 0) {
        for (int kb = kb0; kb < kb1 && kb < kb0 + STAGES; ++kb) {
            tma_prefetch_l2(&tmW, kb * BK, c0);
            if (EPI == kI8Gated) tma_prefetch_l2(&tmW2, kb * BK, c0);
        }
    }
    griddep_wait();
    griddep_launch();

    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % STAGES;
                if (!mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1, p.err, &abort_sh)) {
                    ok = false;
                    break;
                }
                uint8_t *st = smem + s * CF::STAGE;
                mbar_arrive_expect_tx(&full_bar[s], CF::STAGE);
                tma_load_2d(st, &tmW, &full_bar[s], kb * BK, c0);
                if (EPI == kI8Gated)
                    tma_load_2d(st + CF::W_BYTES, &tmW2, &full_bar[s], kb * BK, c0);
                tma_load_2d(st + CF::MATS * CF::W_BYTES, &tmX, &full_bar[s], kb * BK, row0);
            }
            // Its copies have landed before the stages are used for anything else.
            for (int j = std::max(0, it - STAGES); j < it; ++j)
                if (!mbar_wait(&full_bar[j % STAGES], (j / STAGES) & 1, p.err, nullptr)) ok = false;
        }
        __syncwarp();
    } else if (warp == 1) {
        // The whole warp walks the steps and one elected lane issues, so that
        // descriptors and counters stay uniform values.
        constexpr uint32_t IDESC = idesc_i8(BC, T);
        const uint64_t desc = smem_desc(smem_u32(smem), 16, 1024, kLayoutSW128);
        const uint32_t lo = (uint32_t)desc, hi = (uint32_t)(desc >> 32);
        int s = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[s], ph, p.err, &abort_sh));
            if (!ok) break;
            if (elect_one_sync()) {
                const uint32_t dw = lo + s * (CF::STAGE >> 4);
                const uint32_t dx = dw + CF::MATS * (CF::W_BYTES >> 4);
#pragma unroll
                for (int kk = 0; kk < BK / 32; ++kk)
#pragma unroll
                    for (int m = 0; m < CF::MATS; ++m)
                        umma_i8(tmem + m * T, dw + m * (CF::W_BYTES >> 4) + kk * 2, dx + kk * 2,
                                hi, IDESC, kb != kb0 || kk != 0);
                umma_commit(&empty_bar[s]);
            }
            if (++s == STAGES) {
                s = 0;
                ph ^= 1;
            }
        }
        if (elect_one_sync()) umma_commit(&done_bar);
        if (!mbar_wait(&done_bar, 0, p.err, nullptr)) ok = false;
    }
    // Every thread learns whether the products are complete (this also holds the
    // epilogue back until they are).
    ok = __syncthreads_and(ok);
    tc_fence_after();
    int *sums = reinterpret_cast<int *>(smem);  // [MATS][T][BC]
    const int n = (warp & 3) * 32 + lane;       // channel of the tile (epilogue warps)
    const int g = (warp - 2) >> 2;              // warpgroup
    if (warp >= 2 && ok) {
        const uint32_t tbase = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll 1
        for (int c = g * 16; c < CF::MATS * T; c += 32) {
            float v[16];
            tmem_ld16(tbase + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[(c + i) * BC + n] = __float_as_int(v[i]);
        }
        tc_fence_before();
    }
    if (split > 1) cluster_sync();
    else __syncthreads();
    if (warp >= 2 && ok) {
        const int per = T / split, t0 = rank * per;
        const int col = c0 + n;
        const bool in = col < p.N;
        const float ws = in ? ld_global(p.ws + col) : 0.0f;
        const float b = in && p.bias ? ld_global(p.bias + col) : 0.0f;
        float ws2 = 0.0f, b2 = 0.0f;
        if (EPI == kI8Gated && in) {
            ws2 = ld_global(p.ws2 + col);
            if (p.bias2) b2 = ld_global(p.bias2 + col);
        }
        // Rows [t, t + kRows) of the sums m, over the cluster: all loads of a CTA's
        // sums in flight at once.
        auto total = [&](int m, int t, int(&a)[kRows]) {
            const uint32_t at = smem_u32(sums + (m * T + t) * BC + n);
#pragma unroll
            for (int i = 0; i < kRows; ++i) a[i] = 0;
            if (split == 1) {
#pragma unroll
                for (int i = 0; i < kRows; ++i)
                    if (t + i < T) a[i] = sums[(m * T + t + i) * BC + n];
                return;
            }
#pragma unroll 2
            for (int r = 0; r < split; ++r) {
                int v[kRows];
#pragma unroll
                for (int i = 0; i < kRows; ++i) v[i] = t + i < t0 + per ? load_peer(at + i * BC * 4, r) : 0;
#pragma unroll
                for (int i = 0; i < kRows; ++i) a[i] += v[i];
            }
        };
        const int t1 = min(t0 + per, p.M - row0);
        // y = x w^T of rows [t, t + kRows), each as acc * s * w + b.
        auto values8 = [&](int m, int t, float w, float bias, const float(&s)[kRows],
                           float(&y)[kRows]) {
            int a[kRows];
            total(m, t, a);
#pragma unroll
            for (int i = 0; i < kRows; ++i) y[i] = fmaf((float)a[i] * s[i], w, bias);
        };
        auto scales8 = [&](int t, float(&s)[kRows]) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) s[i] = t + i < t1 ? ld_global(p.xs + row0 + t + i) : 0.0f;
        };
        auto store8 = [&](int t, const float(&y)[kRows]) {
            if (!in) return;
#pragma unroll
            for (int i = 0; i < kRows; ++i)
                if (t + i < t1)
                    i8::store1(p.y, p.type, (size_t)(row0 + t + i) * p.ldy + col, y[i],
                                p.accumulate);
        };
        if constexpr (EPI != kI8Heads) {
#pragma unroll 1
            for (int t = t0 + g * kRows; t < t1; t += 2 * kRows) {
                float s[kRows], y[kRows];
                scales8(t, s);
                values8(0, t, ws, b, s, y);
                if (p.act != kI8None) {
#pragma unroll
                    for (int i = 0; i < kRows; i += 2) {
                        const float2 v = i8::act2(make_float2(y[i], y[i + 1]), p.act);
                        y[i] = v.x;
                        y[i + 1] = v.y;
                    }
                }
                if (EPI == kI8Gated) {
                    float u[kRows];
                    values8(1, t, ws2, b2, s, u);
#pragma unroll
                    for (int i = 0; i < kRows; ++i) y[i] *= u[i];
                }
                store8(t, y);
            }
        } else {
            // A tile holds BC / HD whole heads; HD / 32 warps a head.
            float *values = reinterpret_cast<float *>(smem + CF::OFF_VALUES);  // [T][BC]
            float *part = values + T * BC;                                     // [T][4]
            const int head = col / HD, e = n % HD, first = n / HD * (HD / 32);
            const bool rot = head < p.n_q_heads + p.n_kv_heads;
            const float *nw = !rot ? nullptr : head < p.n_q_heads ? p.q_norm : p.k_norm;
            // The other value of this one's rotation, and its sign.
            const int half = HD / 2, pair = e < half ? n + half : n - half;
            const float sign = e < half ? -1.0f : 1.0f;
            const float w1 = nw ? ld_global(nw + e) : 1.0f;
            const float w2 = nw ? ld_global(nw + (e < half ? e + half : e - half)) : 1.0f;
#pragma unroll 1
            for (int t = t0 + g * kRows; t < t1; t += 2 * kRows) {
                float s[kRows], y[kRows], cs[kRows], sn[kRows];
                scales8(t, s);
                uint32_t bad = 0;
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const int ps = rot && t + i < t1 ? ld_global(p.pos + row0 + t + i) : 0;
                    const bool out = ps < 0 || ps >= p.n_pos;
                    bad |= (uint32_t)out << i;
                    const size_t at = (size_t)(out ? 0 : ps) * half + e % half;
                    cs[i] = ld_global(p.cos + at);
                    sn[i] = ld_global(p.sin + at);
                }
                if (bad && in) set_error(p.err, kErrBadPosition);
                values8(0, t, ws, b, s, y);
                if (rot || HD == 64) {  // (a tile of two heads: all of its warps meet)
                    float ss[kRows];
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
                        ss[i] = y[i] * y[i];
                        values[(t + i) % T * BC + n] = y[i];
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                        for (int i = 0; i < kRows; ++i)
                            ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
                    if (lane == 0) {
#pragma unroll
                        for (int i = 0; i < kRows; ++i) part[(t + i) % T * 4 + (warp & 3)] = ss[i];
                    }
                    named_bar(1 + g, 128);
                }
                if (rot) {
#pragma unroll
                    for (int i = 0; i < kRows; ++i) {
                        const int tt = (t + i) % T;
                        float inv = bad >> i & 1 ? i8::nan_f() : 1.0f;
                        if (nw) {
                            float ss = 0.0f;
#pragma unroll
                            for (int k = 0; k < HD / 32; ++k) ss += part[tt * 4 + first + k];
                            inv *= 1.0f / sqrtf(ss / (float)HD + p.eps);
                        }
                        y[i] = i8::rotate(y[i] * inv * w1, values[tt * BC + pair] * inv * w2, cs[i],
                                          sn[i], sign);
                    }
                }
                store8(t, y);
            }
        }
    }
    if (split > 1) cluster_sync();  // no CTA leaves while its sums are read
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, CF::TMEM_COLS);
    }
}

template <int EPI, int T, int HD>
int launch(const I8Params &p, int split, cudaStream_t stream) {
    CUtensorMap mw, mw2, mx;
    constexpr CUtensorMapDataType U8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    constexpr CUtensorMapSwizzle SW = CU_TENSOR_MAP_SWIZZLE_128B;
    if (make_map_ld(&mw, p.w, p.N, p.K, p.ldw, BC, BK, SW, U8, 1) ||
        make_map_ld(&mx, p.x, p.M, p.K, p.ldx, T, BK, SW, U8, 1))
        return -1;
    mw2 = mw;
    if (EPI == kI8Gated && make_map_ld(&mw2, p.w2, p.N, p.K, p.ldw2, BC, BK, SW, U8, 1)) return -1;
    CK((set_smem_once<i8_mid_kernel<EPI, T, HD>>(Cfg<EPI, T>::SMEM)));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((p.N + BC - 1) / BC * split, (p.M + T - 1) / T);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<EPI, T>::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    LAUNCH(cudaLaunchKernelEx(&cfg, i8_mid_kernel<EPI, T, HD>, mw, mw2, mx, p, split));
    return 0;
}

template <int EPI, int HD>
int launch_t(const I8Params &p, int split, cudaStream_t stream) {
    if (p.M <= 16) return launch<EPI, 16, HD>(p, split, stream);
    if (p.M <= 32) return launch<EPI, 32, HD>(p, split, stream);
    if constexpr (EPI != kI8Heads) {
        if (p.M > 64) return launch<EPI, 128, HD>(p, split, stream);
    }
    return launch<EPI, 64, HD>(p, split, stream);
}

// Clusters of `size` CTAs (4 or 8) that the device runs at a time, one CTA to an
// SM: the SMs of a GPC that make up no whole cluster stay idle (here 33 clusters
// of 4 and 15 of 8, not 37 and 18).  One too many costs a second round: 2048
// channels, K = 4096 in 16 clusters of 8 12.0 us, in 16 of 4 6.5 us.
int resident_clusters(int size, int num_sms) {
    static std::atomic<int> known[64][2];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    std::atomic<int> *slot = dev < 64 ? &known[dev][size == 8] : nullptr;
    int n = slot ? slot->load(std::memory_order_relaxed) : 0;
    if (n > 0) return n;
    constexpr auto kern = i8_mid_kernel<kI8Store, 64, 0>;
    constexpr int smem = Cfg<kI8Store, 64>::SMEM;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(num_sms / size * size);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (set_smem_once<kern>(smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        return 0;  // no such clusters: K is split less
    }
    if (slot) slot->store(n, std::memory_order_relaxed);
    return n;
}

}  // namespace

// Channel tiles times row blocks.
long long mid_tiles(int epi, const I8Params &p) {
    const int rows = epi == kI8Heads ? 64 : 128;
    return (p.N + BC - 1ll) / BC * ((p.M + rows - 1) / rows);
}

// Up to 64 rows.  More, where K is long: the 256-row tiles of int8_gemm.cu do
// not split it (4096 channels, K = 12288: 128 rows 14.6 us here, 28.2 there; K =
// 4096: 10.5 and 12.3, K = 2560: 9.6 and 9.3; gate and up of 2048 channels, K =
// 8192: 16.3 and 19.8, of 4096 channels, K = 4096: 14.7 and 13.1).  Heads over 64
// rows, and all over 128, only where the tiles leave SMs to split K over (K =
// 8192, 256 rows: 4096 channels 17.0 and 20.2, 8192 channels 26.3 and 21.3, gate
// and up of 2048 17.5 and 19.7, of 2560 24.3 and 20.1; K = 4096, 128 rows: 12
// heads 10.4 and 14.6, 32 heads 20.5 and 14.8).
bool i8_mid_fits(int epi, const I8Params &p, int num_sms) {
    if (p.M <= 64) return true;
    if (epi == kI8Heads) return p.M <= 128 && p.K >= 2048 && mid_tiles(epi, p) * 4 <= num_sms;
    if (p.M <= 128) return p.K >= (epi == kI8Gated ? 8192 : 4096);
    const int halves = epi == kI8Gated ? 4 : 2;
    return p.M <= 256 && p.K >= 8192 && mid_tiles(epi, p) * halves <= num_sms;
}

int i8_mid_run(int epi, const I8Params &p, int num_sms, cudaStream_t stream) {
    // K is split while all clusters run at a time and each CTA keeps two steps;
    // in eight, only where it keeps 4 (up to 32 rows; 1024 channels, K = 4096:
    // 6.2 us against 6.5 of four, K = 2560: 6.0 and 5.6) or 8 (1024 channels, 64
    // rows, K = 4096: 7.9 and 7.4, K = 12288: 10.1 and 11.0).
    const long long tiles = mid_tiles(epi, p);
    const int k_blocks = (p.K + BK - 1) / BK;
    int split = 1;
    for (int c = 2; c <= 8; c *= 2) {
        const int steps = c < 8 ? 2 : p.M <= 32 ? 4 : 8;
        if (tiles * c > num_sms || k_blocks < steps * c) break;
        if (c > 2 && tiles > resident_clusters(c, num_sms)) break;
        split = c;
    }
    switch (epi) {
    case kI8Store: return launch_t<kI8Store, 0>(p, split, stream);
    case kI8Gated: return launch_t<kI8Gated, 0>(p, split, stream);
    case kI8Heads:
        return p.head_dim == 128 ? launch_t<kI8Heads, 128>(p, split, stream)
                                 : launch_t<kI8Heads, 64>(p, split, stream);
    }
    return -1;
}

}  // namespace fb
