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
// columns meet in one accumulator.  Bound by the tensor cores at the clock that
// the power cap leaves and the 64 KB a pair takes from L2 per 128 bytes of K
// (12.8 TB/s over all SMs), at short K by the epilogue.  Measured: 8192 x 4096 x
// 12288 254 us (3.2 POPS), gate and up 8192 x 12288 x 4096 485 us (3.4), 8192 x
// 4096 x 1024 31 us, with GELU 39.5 us, heads of 32768 x 4096 x 1024 145 us, of
// 8192 x 6144 x 4096 143 us.
//
// Roles per CTA: warp 0 TMA producer, warp 1 TMEM allocation and (leader) MMA
// issue, the other warps the epilogue, in warpgroups that split the columns.  No
// TMA load uses multicast.
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
constexpr int A_BYTES = BM * BK;
constexpr int CHUNK = 2048;   // 32 rows x 64 bytes of output
constexpr uint32_t kPeerMask = 0xFEFFFFFFu;  // clears the CTA-rank bit: leader's copy

// Shared memory: the stages, 2 KB of output per epilogue warp and, in the head
// form, the rotary rows of the CTA's 128 rows (cos and sin, f32, each row
// padded by 16 bytes so that 32 lanes reading 16 bytes of a row each meet no
// bank twice).  Stores from registers would touch 32 rows an instruction (60
// cycles of the shared-memory pipe each, 3000 a tile).  The head form and the
// gated form have two epilogue warpgroups (a thread holds a whole head, or 32
// gate and 32 up sums), the plain one four.
template <int BN, int EPI, int HD>
struct Cfg {
    static constexpr bool HEADS = EPI == kI8Heads;
    static constexpr int B_BYTES = (BN / 2) * BK;  // this CTA's half of the weight rows
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = HEADS ? (BN == 256 ? 4 : 5) : BN == 256 ? 5 : BN == 128 ? 7 : 8;
    static constexpr int OFF_STAGING = STAGES * STAGE;
    static constexpr int GROUPS = EPI == kI8Store ? 4 : 2;  // epilogue warpgroups
    static constexpr int THREADS = 64 + 128 * GROUPS;
    static constexpr int ROPE_LD = HD + 4;  // floats
    static constexpr int OFF_ROPE = OFF_STAGING + 4 * GROUPS * CHUNK;
    // Per warpgroup, twice: the scales and biases of its columns of the tile.
    static constexpr int MIN_COLS = EPI == kI8Gated ? 64 : 32;  // of one unit
    static constexpr int GCOLS = HEADS ? 128 : BN / GROUPS < MIN_COLS ? MIN_COLS : BN / GROUPS;
    static constexpr int OFF_COLS = OFF_ROPE + (HEADS ? BM * ROPE_LD * 4 : 0);
    static constexpr int OFF_NORMS = OFF_COLS + GROUPS * 2 * 2 * GCOLS * 4;
    static constexpr int SMEM = OFF_NORMS + (HEADS ? 2 * HD * 4 : 0) + 1024;
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

// D[tmem, s32] (+)= A * B^T, 8-bit integers; the operands' descriptors share
// their upper word.
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                             uint32_t hi, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accum)
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

// Arrive on the leader CTA's copy of `bar`.  It hands over TMEM that this
// thread's completed loads have read, no memory: a release at cluster scope
// would wait for the thread's earlier stores (measured at 1500 cycles a tile).
__device__ __forceinline__ void arrive_leader(uint64_t *bar) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(smem_u32(bar)));
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}

// Neighbouring values packed in the 16-bit type (one branch for all of them).
template <int N>
__device__ __forceinline__ void pack32(uint32_t (&w)[N], const float (&v)[2 * N], bool f16) {
    if (f16) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = pack_f16x2(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    }
}

// Output of one warp (32 rows): 64-byte row segments (32 16-bit or 16 f32
// columns) staged in shared memory with the 64-byte swizzle, then one TMA store
// (or f32 reduce-add) per chunk, so a warp waits for no other; where the
// output's base or row stride is not a multiple of 16 bytes, the warp writes
// the chunk's elements itself, a row segment at a time.  Rows past M and
// columns past N are left alone.
struct Sink {
    const I8Params &p;
    const CUtensorMap *map;
    uint8_t *stage;  // one chunk
    int lane, y0;    // y0: first row
    bool tma;

    __device__ __forceinline__ uint8_t *acquire() {
        if (lane == 0 && tma) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
        return stage;
    }
    __device__ __forceinline__ void publish(uint8_t *buf, int col) {
        if (tma) fence_proxy_async_smem();
        __syncwarp();
        if (tma) {
            if (lane == 0) {
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
            const bool f32 = p.type == kI8F32;
            const int c = lane & (f32 ? 15 : 31);
            const int byte = f32 ? c * 4 : c * 2;
            if (col + c < p.N) {
                const int rows = min(32, p.M - y0);
                for (int i = f32 ? lane >> 4 : 0; i < rows; i += f32 ? 2 : 1) {
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
                    *reinterpret_cast<float4 *>(buf + lane * 64 + ((c ^ ((lane >> 1) & 3)) * 16)) =
                        make_float4(v[16 * h + 4 * c], v[16 * h + 4 * c + 1],
                                    v[16 * h + 4 * c + 2], v[16 * h + 4 * c + 3]);
                publish(buf, col + 16 * h);
            }
            return;
        }
        uint32_t w[16];
        pack32(w, v, p.type == kI8F16);
        uint8_t *buf = acquire();
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4 *>(buf + lane * 64 + ((c ^ ((lane >> 1) & 3)) * 16)) =
                make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
        publish(buf, col);
    }
    __device__ __forceinline__ void finish() {
        if (lane == 0 && tma) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
};

// 32 integer sums (as bits) scaled: v = v * s * t + b (b null: no bias).  (The
// conversion instruction is slow but runs beside the arithmetic; conversions by
// adding 1.5 x 2^23 to the bits, with a check of their range, measured 10-20 %
// slower in the gated form.)
__device__ __forceinline__ void scale32(float (&v)[32], float s, const float *t, const float *b) {
    const float2 s2 = make_float2(s, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 tv = reinterpret_cast<const float4 *>(t)[i];
        float4 bv = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (b) bv = reinterpret_cast<const float4 *>(b)[i];
        const float2 a0 = mul_f32x2(make_float2((float)__float_as_int(v[4 * i]),
                                                (float)__float_as_int(v[4 * i + 1])),
                                    s2);
        const float2 a1 = mul_f32x2(make_float2((float)__float_as_int(v[4 * i + 2]),
                                                (float)__float_as_int(v[4 * i + 3])),
                                    s2);
        const float2 r0 = fma_f32x2(a0, make_float2(tv.x, tv.y), make_float2(bv.x, bv.y));
        const float2 r1 = fma_f32x2(a1, make_float2(tv.z, tv.w), make_float2(bv.z, bv.w));
        v[4 * i] = r0.x;
        v[4 * i + 1] = r0.y;
        v[4 * i + 2] = r1.x;
        v[4 * i + 3] = r1.y;
    }
}

template <typename F>
__device__ __forceinline__ void pairs(float (&v)[32], F f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 r = f(make_float2(v[2 * i], v[2 * i + 1]));
        v[2 * i] = r.x;
        v[2 * i + 1] = r.y;
    }
}

__device__ __forceinline__ void act32(float (&v)[32], int act) {
    if (act == kI8None) return;
    if (act == kI8Silu) pairs(v, i8::silu);
    else if (act == kI8GeluErf) pairs(v, i8::gelu_erf);
    else pairs(v, i8::gelu_tanh);
}

// Column of the tile's accumulator behind entry j of a warpgroup's column table
// (its units of 32 columns, gate and up for the gated form, or its heads).
template <int BN, int EPI, int HD, int G>
__device__ __forceinline__ int table_col(int g, int j) {
    if (EPI == kI8Store) return (g + j / 32 * G) * 32 + j % 32;
    if (EPI == kI8Gated) return j / 32 % 2 * (BN / 2) + (g + j / 64 * G) * 32 + j % 32;
    return (g + j / (HD ? HD : 1) * G) * HD + j % (HD ? HD : 1);
}

// One 128-row x BN accumulator; a warpgroup takes every G-th unit of 32 output
// columns.  cols: the scales, then (NC on) the biases of its columns.  release
// is called once the accumulator has been read.
template <int BN, int EPI, int G, int NC, typename F>
__device__ __forceinline__ void epilogue(const I8Params &p, uint32_t tbase, float s, int nb, int g,
                                         const float *cols, Sink &sink, F release) {
    const float *bias = p.bias ? cols + NC : nullptr;
    if constexpr (EPI == kI8Store) {
        constexpr int UNITS = NC / 32;
#pragma unroll 1
        for (int u = 0; u < UNITS; ++u) {
            const int c = (g + u * G) * 32;
            const bool in = c < BN && nb * BN + c < p.N;
            float v[32];
            if (in) {
                tmem_ld32(tbase + c, v);
                tmem_wait_ld();
            }
            if (u == UNITS - 1) release();
            if (!in) continue;
            scale32(v, s, cols + u * 32, bias ? bias + u * 32 : nullptr);
            act32(v, p.act);
            sink.put(v, nb * BN + c);
        }
    } else {
        constexpr int UNITS = NC / 64;
#pragma unroll 1
        for (int k = 0; k < UNITS; ++k) {
            const int c = (g + k * G) * 32, col = nb * (BN / 2) + c;
            const bool in = c < BN / 2 && col < p.N;
            float v[2][32];  // gate, up
            if (in) {
                tmem_ld32(tbase + c, v[0]);
                tmem_ld32(tbase + BN / 2 + c, v[1]);
                tmem_wait_ld();
            }
            if (k == UNITS - 1) release();
            if (!in) continue;
            scale32(v[0], s, cols + k * 64, bias ? bias + k * 64 : nullptr);
            act32(v[0], p.act);
            scale32(v[1], s, cols + k * 64 + 32, p.bias2 ? cols + NC + k * 64 + 32 : nullptr);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[0][i] *= v[1][i];
            sink.put(v[0], col);
        }
    }
}

// The head form: a warpgroup takes every second head of the tile.  A thread
// holds its row's whole head in registers, so TMEM is read once.  rope: the
// row's cos and sin [HD / 2] each (shared memory); norms: q_norm, k_norm [HD].
template <int BN, int HD, int G, int NC, typename F>
__device__ __forceinline__ void epilogue_heads(const I8Params &p, uint32_t tbase, float s, bool bad,
                                               int nb, int g, const float *cols,
                                               const float *rope, const float *norms, Sink &sink,
                                               F release) {
    constexpr int HALF = HD / 2, H32 = HALF / 32;
    const float *bias = p.bias ? cols + NC : nullptr;
    if (g * HD >= BN || nb * BN + g * HD >= p.N) {
        release();
        return;
    }
#pragma unroll 1
    for (int h0 = g * HD, k = 0; h0 < BN; h0 += G * HD, ++k) {
        const int col0 = nb * BN + h0;
        if (col0 >= p.N) break;
        const int head = col0 / HD;
        const bool is_q = head < p.n_q_heads;
        const bool rot = head < p.n_q_heads + p.n_kv_heads;
        float v[HD / 32][32];
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) tmem_ld32(tbase + h0 + c * 32, v[c]);
        tmem_wait_ld();
        if (h0 + G * HD >= BN || col0 + G * HD >= p.N) release();  // the last head
#pragma unroll
        for (int c = 0; c < HD / 32; ++c)
            scale32(v[c], s, cols + k * HD + c * 32, bias ? bias + k * HD + c * 32 : nullptr);
        if (rot) {
            const bool normed = is_q ? p.q_norm != nullptr : p.k_norm != nullptr;
            float inv = bad ? i8::nan_f() : 1.0f;
            if (normed) {
                float2 q[4] = {};
#pragma unroll
                for (int c = 0; c < HD / 32; ++c)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 x = make_float2(v[c][2 * i], v[c][2 * i + 1]);
                        q[i & 3] = fma_f32x2(x, x, q[i & 3]);
                    }
                const float2 t = add_f32x2(add_f32x2(q[0], q[1]), add_f32x2(q[2], q[3]));
                inv *= 1.0f / sqrtf((t.x + t.y) / (float)HD + p.eps);
            }
            const float *nw = norms + (is_q ? 0 : HD);
            const float2 inv2 = make_float2(inv, inv);
#pragma unroll
            for (int c = 0; c < H32; ++c) {
                float(&A)[32] = v[c], (&B)[32] = v[H32 + c];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = c * 8 + i;
                    const float4 cv = reinterpret_cast<const float4 *>(rope)[e];
                    const float4 sv = reinterpret_cast<const float4 *>(rope + HALF)[e];
                    float4 w1 = make_float4(1.0f, 1.0f, 1.0f, 1.0f), w2 = w1;
                    if (normed) {
                        w1 = reinterpret_cast<const float4 *>(nw)[e];
                        w2 = reinterpret_cast<const float4 *>(nw + HALF)[e];
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int j = 4 * i + 2 * u;
                        const float2 c2 = u ? make_float2(cv.z, cv.w) : make_float2(cv.x, cv.y);
                        const float2 s2 = u ? make_float2(sv.z, sv.w) : make_float2(sv.x, sv.y);
                        float2 a = mul_f32x2(make_float2(A[j], A[j + 1]), inv2);
                        float2 b = mul_f32x2(make_float2(B[j], B[j + 1]), inv2);
                        if (normed) {
                            a = mul_f32x2(a, u ? make_float2(w1.z, w1.w) : make_float2(w1.x, w1.y));
                            b = mul_f32x2(b, u ? make_float2(w2.z, w2.w) : make_float2(w2.x, w2.y));
                        }
                        // (as i8::rotate)
                        const float2 r1 = mul_f32x2(a, c2);
                        const float2 r2 = fma_f32x2(a, s2, mul_f32x2(b, c2));
                        A[j] = fmaf(-b.x, s2.x, r1.x);
                        A[j + 1] = fmaf(-b.y, s2.y, r1.y);
                        B[j] = r2.x;
                        B[j + 1] = r2.y;
                    }
                }
                sink.put(A, col0 + c * 32);
                sink.put(B, col0 + HALF + c * 32);
            }
        } else {
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) sink.put(v[c], col0 + c * 32);
        }
    }
}

// Tiles of one SM pair, in order.  The pairs take turns over groups of row
// blocks, columns outermost within a group: the pairs' tiles of one moment then
// share both operands (with row blocks outermost they would share one row block
// and read 74 different weight tiles, all of a large matrix per row block).  A
// group is 8 blocks.  Gate and up weights that do not stay in L2 are read once a
// group, so there it is as many as 32 MB of quantised rows allow, up to 32 (8192 x
// 12288 x 4096 with 8 and 32 blocks 510 and 485 us, 32768 rows of it 2210 and
// 2120; plain products of 4096 columns lose 1-2 % by larger groups).
// Head form, K <= kRunK: a pair takes a run of neighbouring tiles, row blocks
// outermost, so that the rotary rows, 3000 cycles to fetch, change seldom; but
// the pairs are then at 74 places of the weights and hold 74 row blocks, which L2
// keeps only while K is short, and a longer K hides the rows' fetch.  Heads in
// runs and in turns: 32768 x 4096 x 1024 146 and 189 us, 32768 x 6144 x 2048 309
// and 340, 8192 x 6144 x 2560 94 and 97, 32768 x 6144 x 2560 400 and 364, 16384 x
// 6144 x 4096 380 and 278, 16384 x 7168 x 5120 580 and 411.
constexpr int kRaster = 8;
constexpr int kRunK = 2048;
constexpr long long kKeptWeights = 24ll << 20;  // bytes

int raster_group(const I8Params &p) {
    if (2ll * p.N * p.K <= kKeptWeights) return kRaster;
    return (int)std::max<long long>(kRaster, std::min(32ll, (32ll << 20) / (2ll * BM * p.K)));
}

// (What the launch's parameters give is computed anew: the head form's epilogue
// has no registers left to keep it in.)
template <int EPI, int TN>
struct Tiles {
    const I8Params &p;
    const int &group_rows;
    int next, end;
    __device__ __forceinline__ int m_blocks() const { return (p.M + 2 * BM - 1) / (2 * BM); }
    __device__ __forceinline__ int n_blocks() const { return (p.N + TN - 1) / TN; }
    __device__ __forceinline__ int pairs() const { return gridDim.x >> 1; }
    __device__ __forceinline__ bool runs() const { return EPI == kI8Heads && p.K <= kRunK; }
    __device__ Tiles(const I8Params &p_, const int &group_rows_) : p(p_), group_rows(group_rows_) {
        const int total = m_blocks() * n_blocks(), pair = blockIdx.x >> 1;
        next = runs() ? (int)((long long)total * pair / pairs()) : pair;
        end = runs() ? (int)((long long)total * (pair + 1) / pairs()) : total;
    }
    __device__ __forceinline__ bool pop(int &mb, int &nb) {
        if (next >= end) return false;
        if (runs()) {
            mb = next / n_blocks();
            nb = next % n_blocks();
            ++next;
        } else {
            const int R = EPI == kI8Gated ? group_rows : kRaster;
            const int group = next / (R * n_blocks());
            const int rows = min(R, m_blocks() - group * R);
            const int r = next - group * R * n_blocks();
            mb = group * R + r % rows;
            nb = r / rows;
            next += pairs();
        }
        return true;
    }
};

template <int BN, int EPI, int HD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__((Cfg<BN, EPI, HD>::THREADS), 1)
    i8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmB2,
                   const __grid_constant__ CUtensorMap tmOut, const I8Params p, const int tma_out,
                   const int group_rows) {
    extern __shared__ uint8_t smem_raw[];
    using CF = Cfg<BN, EPI, HD>;
    constexpr int STAGES = CF::STAGES, GROUPS = CF::GROUPS;
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
    const int k_blocks = (p.K + BK - 1) / BK;
    Tiles<EPI, TN> tiles(p, group_rows);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull_bar[a], 1);
            mbar_init(&tempty_bar[a], 2 * 4 * GROUPS);
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
            int mb, nb;
            while (ok && tiles.pop(mb, nb)) {
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
        if (leader) {
            // ---------------------------------------------------------- MMA issuer
            // The whole warp walks the steps and one elected lane issues, so that
            // descriptors and counters stay uniform values.  This thread's
            // instructions set the pace of long products: with a lone lane in the
            // loop, and descriptors built anew for every product, a step of K took
            // 609 cycles instead of 580 (512 are the tensor cores').
            constexpr uint32_t IDESC = idesc_i8(2 * BM, BN);
            const uint64_t desc = smem_desc(smem_u32(smem), 16, 1024, kLayoutSW128);
            const uint32_t lo = (uint32_t)desc, hi = (uint32_t)(desc >> 32);
            int lt = 0, s = 0;
            uint32_t ph = 0;
            bool ok = true;
            int mb, nb;
            for (; ok && tiles.pop(mb, nb); ++lt) {
                const int a = lt & 1;
                const uint32_t aph = (lt >> 1) & 1;
                ok = __all_sync(0xffffffffu, mbar_wait(&tempty_bar[a], aph ^ 1, p.err, &abort_sh));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem_base + a * BN;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[s], ph, p.err, &abort_sh));
                    if (!ok) break;
                    if (elect_one_sync()) {
                        const uint32_t da = lo + s * (CF::STAGE >> 4), db = da + (A_BYTES >> 4);
#pragma unroll
                        for (int kk = 0; kk < BK / 32; ++kk)
                            umma_i8_pair(d, da + kk * 2, db + kk * 2, hi, IDESC, (kb | kk) != 0);
                        umma_commit_pair(&empty_bar[s]);
                    }
                    if (++s == STAGES) {
                        s = 0;
                        ph ^= 1;
                    }
                }
                if (!ok) break;
                if (elect_one_sync()) umma_commit_pair(&tfull_bar[a]);
            }
            if (!ok) {
                if (elect_one_sync())
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
        const int et = (warp - 2) * 32 + lane;          // thread of the epilogue
        constexpr int NC = CF::GCOLS, LOADS = (2 * NC + 127) / 128;
        float *cols0 = reinterpret_cast<float *>(smem + CF::OFF_COLS) + g * 4 * NC;
        Sink sink{p, &tmOut, smem + CF::OFF_STAGING + (warp - 2) * CHUNK, lane, 0, tma_out != 0};
        float *rope = reinterpret_cast<float *>(smem + CF::OFF_ROPE);
        float *norms = reinterpret_cast<float *>(smem + CF::OFF_NORMS);
        if (EPI == kI8Heads) {
            for (int i = et; i < HD; i += 128 * GROUPS) {
                norms[i] = p.q_norm ? ld_global(p.q_norm + i) : 1.0f;
                norms[HD + i] = p.k_norm ? ld_global(p.k_norm + i) : 1.0f;
            }
        }
        // A tile's row scale, column scales and biases are fetched one tile
        // ahead; the columns' go through two buffers in shared memory (a thread
        // writes one after a barrier that all of its last readers have passed).
        float s_next = 0.0f, c_next[LOADS];
        auto fetch = [&](int mb, int nb) {
            const int grow = mb * 2 * BM + (int)rank * BM + row;
            s_next = grow < p.M ? ld_global(p.xs + grow) : 0.0f;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int e = gt + i * 128;
                c_next[i] = 0.0f;
                if (e >= 2 * NC) break;
                const int c = table_col<BN, EPI, HD, GROUPS>(g, e % NC);
                const bool second = EPI == kI8Gated && c >= TN;
                const int col = nb * TN + (second ? c - TN : c);
                const float *src = e < NC ? (second ? p.ws2 : p.ws) : (second ? p.bias2 : p.bias);
                if (src && c < BN && col < p.N) c_next[i] = ld_global(src + col);
            }
        };
        auto keep = [&](float *cols) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                if (gt + i * 128 < 2 * NC) cols[gt + i * 128] = c_next[i];
        };
        int lt = 0, mb = 0, nb = 0, rope_mb = -1;
        bool bad = false, more = tiles.pop(mb, nb);
        if (more) {
            fetch(mb, nb);
            keep(cols0);
        }
        for (; more; ++lt) {
            const int a = lt & 1;
            const uint32_t aph = (lt >> 1) & 1;
            const int mb0 = mb, nb0 = nb;
            const int y0 = mb0 * 2 * BM + (int)rank * BM;
            const int grow = y0 + row;
            const float s = s_next;
            float *cols = cols0 + a * 2 * NC;
            more = tiles.pop(mb, nb);
            if (more) fetch(mb, nb);
            if constexpr (EPI == kI8Heads) {
                if (mb0 != rope_mb) {
                    // The rotary rows of this row block: a warp copies 16 rows,
                    // eight loads before their stores (32768 x 4096 x 1024 heads
                    // 153 us, one at a time 168).  All warps are past their last reads.
                    rope_mb = mb0;
                    named_bar(1 + GROUPS, 128 * GROUPS);
                    const int ps = grow < p.M ? ld_global(p.pos + grow) : 0;
                    bad = ps < 0 || ps >= p.n_pos;
                    if (bad) set_error(p.err, kErrBadPosition);
                    constexpr int V = HD / 4;  // float4 per row, cos then sin
#pragma unroll
                    for (int i0 = 0; i0 < 16; i0 += 8) {
                        float4 v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            int rp = __shfl_sync(0xffffffffu, ps, g * 16 + i0 + i);
                            if (rp < 0 || rp >= p.n_pos) rp = 0;
                            const float *src =
                                (lane % V < V / 2 ? p.cos : p.sin) + (size_t)rp * (HD / 2);
                            v[i] = ld_global(reinterpret_cast<const float4 *>(src) + lane % (V / 2));
                        }
                        if (lane < V) {
                            const int r = q * 32 + g * 16 + i0;
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                reinterpret_cast<float4 *>(rope + (r + i) * CF::ROPE_LD)[lane] = v[i];
                        }
                    }
                    named_bar(1 + GROUPS, 128 * GROUPS);
                }
            }
            // One verdict for the warpgroup (its barriers need all of it), and
            // in the head form for both.
            const bool ok = mbar_wait(&tfull_bar[a], aph, p.err, &abort_sh);
            if (!(EPI == kI8Heads ? named_bar_and(1 + GROUPS, 128 * GROUPS, ok)
                                  : named_bar_and(1 + g, 128, ok)))
                break;
            tc_fence_after();
            const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + a * BN;
            auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_leader(&tempty_bar[a]);
            };
            sink.y0 = y0 + q * 32;
            if (sink.y0 >= p.M)
                release();
            else if constexpr (EPI == kI8Heads)
                epilogue_heads<BN, HD, GROUPS, NC>(p, tbase, s, bad, nb0, g, cols,
                                                   rope + row * CF::ROPE_LD, norms, sink, release);
            else
                epilogue<BN, EPI, GROUPS, NC>(p, tbase, s, nb0, g, cols, sink, release);
            if (more) keep(cols0 + (a ^ 1) * 2 * NC);
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
    if (tma && make_map_ld(&mo, p.y, p.M, p.N, p.ldy, 32, 64 / esz, CU_TENSOR_MAP_SWIZZLE_64B,
                           p.type == kI8F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                           : p.type == kI8BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           esz))
        return -1;
    CK((set_smem_once<i8_gemm_kernel<BN, EPI, HD>>(Cfg<BN, EPI, HD>::SMEM)));
    constexpr int TN = EPI == kI8Gated ? BN / 2 : BN;
    const long long tiles = (long long)((p.M + 2 * BM - 1) / (2 * BM)) * ((p.N + TN - 1) / TN);
    const int grid = (int)std::min<long long>(2 * tiles, num_sms & ~1);
    LAUNCH(launch_k(i8_gemm_kernel<BN, EPI, HD>, dim3(grid), dim3(Cfg<BN, EPI, HD>::THREADS), (Cfg<BN, EPI, HD>::SMEM), stream,
                    ma, mb, mb2, mo, p, tma ? 1 : 0,
                    EPI == kI8Gated ? raster_group(p) : kRaster));
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
