// C entry points of the 8-bit integer projections (include/ffwd_b200.h).
#include "ffwd_b200.h"
#include "host_util.h"
#include "int8.cuh"

#include <cmath>

namespace fb {
namespace {

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// A kernel that is handed another GPU's or the host's pageable memory would
// fault: such pointers are refused here.
int check_device(const char *name, const void *ptr, int dev) {
    if (!ptr) return 0;
    cudaPointerAttributes at{};
    CK(cudaPointerGetAttributes(&at, ptr));
    if (at.type != cudaMemoryTypeManaged && !(at.type == cudaMemoryTypeDevice && at.device == dev)) {
        fail("%s is not memory of the current device %d", name, dev);
        return -1;
    }
    return 0;
}

int device_info(int *dev, int *sms) {
    CK(cudaGetDevice(dev));
    CK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *dev));
    return 0;
}

// Rows of one call: tile arithmetic stays within 32 bits.
constexpr int kMaxRows = 1 << 30;

bool type_ok(int t) { return t == kI8F32 || t == kI8BF16 || t == kI8F16; }

// Shapes, strides and alignment of the quantised rows.  (No rows: a tensor
// without elements has no address.)
int check_rows(const int8_t *x, long long ldx, const float *xs, int M, int K) {
    if (M < 0 || M > kMaxRows || (M > 0 && (!x || !xs))) {
        fail("invalid arguments");
        return -1;
    }
    if (!aligned16(x) || ldx % 16 || ldx < K) {
        fail("int8 rows need a 16-byte aligned base and a row stride of at least %d, a multiple "
             "of 16 (got %lld)",
             K, ldx);
        return -1;
    }
    if (!aligned4(xs)) {
        fail("scales need 4-byte alignment");
        return -1;
    }
    return 0;
}

int check_mat(const ffwd_b200_i8_mat_t *w) {
    if (!w || !w->q || !w->scale || w->rows <= 0 || w->rows > kMaxRows || w->cols <= 0) {
        fail("invalid weights");
        return -1;
    }
    if (w->cols > kI8MaxK) {
        fail("%d columns: 32-bit sums of int8 products hold at most %d", w->cols, kI8MaxK);
        return -1;
    }
    if (!aligned16(w->q) || w->ld % 16 || w->ld < w->cols) {
        fail("int8 weights need a 16-byte aligned base and a row stride of at least %d, a "
             "multiple of 16 (got %lld)",
             w->cols, w->ld);
        return -1;
    }
    if (!aligned4(w->scale) || !aligned4(w->bias)) {
        fail("scales and biases need 4-byte alignment");
        return -1;
    }
    return 0;
}

int check_out(const void *y, int type, long long ldy, int M, int N) {
    if ((M > 0 && !y) || !type_ok(type)) {
        fail("invalid arguments");
        return -1;
    }
    const uintptr_t esz = type == kI8F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(y) % esz || ldy < N) {
        fail("output needs element alignment and a row stride of at least %d (got %lld)", N, ldy);
        return -1;
    }
    return 0;
}

int run(int epi, const I8Params &p, const float *const (&extra)[4], cudaStream_t stream) {
    if (!aligned4(p.err)) {
        fail("the error word needs 4-byte alignment");
        return -1;
    }
    if (p.M == 0) return 0;
    int dev = 0, sms = 148;
    if (device_info(&dev, &sms)) return -1;
    if (check_device("x", p.x, dev) || check_device("x scales", p.xs, dev) ||
        check_device("weights", p.w, dev) || check_device("weight scales", p.ws, dev) ||
        check_device("bias", p.bias, dev) || check_device("weights", p.w2, dev) ||
        check_device("weight scales", p.ws2, dev) || check_device("bias", p.bias2, dev) ||
        check_device("output", p.y, dev) || check_device("error word", p.err, dev) ||
        check_device("positions", p.pos, dev))
        return -1;
    for (const float *e : extra)
        if (check_device("head tables", e, dev)) return -1;
    return i8_project(epi, p, sms, stream);
}

void set_mat(I8Params &p, const ffwd_b200_i8_mat_t *w) {
    p.N = w->rows;
    p.K = w->cols;
    p.w = w->q;
    p.ws = w->scale;
    p.bias = w->bias;
    p.ldw = w->ld;
}

}  // namespace

int i8_project(int epi, const I8Params &p, int num_sms, cudaStream_t stream) {
    if (i8_vec_fits(epi, p)) {
        LAUNCH(i8_vec_launch(epi, p, num_sms, stream));
        return 0;
    }
    if (i8_mid_fits(epi, p, num_sms)) return i8_mid_run(epi, p, num_sms, stream);
    return i8_gemm_run(epi, p, num_sms, stream);
}

}  // namespace fb

using namespace fb;

extern "C" {

FFWD_B200_API int ffwd_b200_quantize_i8(const void *x, int type, long long ldx, const float *norm,
                                        float eps, int8_t *q, long long ldq, float *scale, int M,
                                        int K, void *stream) {
    clear_error();
    if ((M > 0 && (!x || !q || !scale)) || !type_ok(type) || M < 0 || M > kMaxRows || K <= 0 ||
        K > kMaxRows) {
        fail("invalid arguments");
        return -1;
    }
    const uintptr_t esz = type == kI8F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % esz || ldx < K) {
        fail("rows need element alignment and a stride of at least %d (got %lld)", K, ldx);
        return -1;
    }
    if (!aligned16(q) || ldq % 16 || ldq < K) {
        fail("int8 rows need a 16-byte aligned base and a row stride of at least %d, a multiple "
             "of 16 (got %lld)",
             K, ldq);
        return -1;
    }
    if (!aligned4(scale) || !aligned4(norm)) {
        fail("scales and norm weights need 4-byte alignment");
        return -1;
    }
    if (norm && !(eps > 0.0f && std::isfinite(eps))) {
        fail("the norm needs a positive eps");
        return -1;
    }
    if (M == 0) return 0;
    int dev = 0, sms = 148;
    if (device_info(&dev, &sms)) return -1;
    if (check_device("x", x, dev) || check_device("norm weights", norm, dev) ||
        check_device("output", q, dev) || check_device("scales", scale, dev))
        return -1;
    LAUNCH(i8_quantize_launch(x, type, ldx, norm, eps, q, ldq, scale, M, K, sms,
                              static_cast<cudaStream_t>(stream)));
    return 0;
}

FFWD_B200_API int ffwd_b200_gemm_i8(const ffwd_b200_i8_mat_t *w, const int8_t *x, long long ldx,
                                    const float *xs, int M, void *y, int type, long long ldy,
                                    int act, int accumulate, int *err, void *stream) {
    clear_error();
    if (check_mat(w) || check_rows(x, ldx, xs, M, w->cols) || check_out(y, type, ldy, M, w->rows))
        return -1;
    if (act < kI8None || act > kI8GeluTanh) {
        fail("unknown activation %d", act);
        return -1;
    }
    if (accumulate && type != kI8F32) {
        fail("only f32 output accumulates");
        return -1;
    }
    I8Params p{};
    p.M = M;
    set_mat(p, w);
    p.x = x;
    p.ldx = ldx;
    p.xs = xs;
    p.y = y;
    p.type = type;
    p.ldy = ldy;
    p.act = act;
    p.accumulate = accumulate != 0;
    p.err = err;
    return run(kI8Store, p, {}, static_cast<cudaStream_t>(stream));
}

FFWD_B200_API int ffwd_b200_gated_i8(const ffwd_b200_i8_mat_t *gate, const ffwd_b200_i8_mat_t *up,
                                     const int8_t *x, long long ldx, const float *xs, int M,
                                     void *h, int type, long long ldh, int act, int *err,
                                     void *stream) {
    clear_error();
    if (check_mat(gate) || check_mat(up)) return -1;
    if (gate->rows != up->rows || gate->cols != up->cols) {
        fail("gate is %d x %d, up %d x %d", gate->rows, gate->cols, up->rows, up->cols);
        return -1;
    }
    if (check_rows(x, ldx, xs, M, gate->cols) || check_out(h, type, ldh, M, gate->rows)) return -1;
    if (act < kI8Silu || act > kI8GeluTanh) {
        fail("unknown gate activation %d", act);
        return -1;
    }
    I8Params p{};
    p.M = M;
    set_mat(p, gate);
    p.w2 = up->q;
    p.ws2 = up->scale;
    p.bias2 = up->bias;
    p.ldw2 = up->ld;
    p.x = x;
    p.ldx = ldx;
    p.xs = xs;
    p.y = h;
    p.type = type;
    p.ldy = ldh;
    p.act = act;
    p.err = err;
    return run(kI8Gated, p, {}, static_cast<cudaStream_t>(stream));
}

FFWD_B200_API int ffwd_b200_qkv_i8(const ffwd_b200_i8_mat_t *w, const ffwd_b200_i8_heads_t *heads,
                                   const int8_t *x, long long ldx, const float *xs, int M,
                                   void *out, int type, long long ldo, int *err, void *stream) {
    clear_error();
    if (check_mat(w)) return -1;
    if (!heads || heads->n_heads <= 0 || heads->n_kv_heads <= 0 || heads->n_pos <= 0 ||
        (M > 0 && !heads->pos) || !heads->cos || !heads->sin) {
        fail("invalid heads");
        return -1;
    }
    if (heads->head_dim != 64 && heads->head_dim != 128) {
        fail("head_dim %d unsupported (64 or 128)", heads->head_dim);
        return -1;
    }
    if (((long long)heads->n_heads + 2ll * heads->n_kv_heads) * heads->head_dim != w->rows) {
        fail("%d query and %d key/value heads of %d do not make %d rows", heads->n_heads,
             heads->n_kv_heads, heads->head_dim, w->rows);
        return -1;
    }
    if ((heads->q_norm || heads->k_norm) && !(heads->eps > 0.0f && std::isfinite(heads->eps))) {
        fail("the head norms need a positive eps");
        return -1;
    }
    if (!aligned16(heads->cos) || !aligned16(heads->sin) || !aligned16(heads->q_norm) ||
        !aligned16(heads->k_norm) || !aligned4(heads->pos)) {
        fail("rotary tables and head norms need 16-byte alignment");
        return -1;
    }
    if (check_rows(x, ldx, xs, M, w->cols) || check_out(out, type, ldo, M, w->rows)) return -1;
    I8Params p{};
    p.M = M;
    set_mat(p, w);
    p.x = x;
    p.ldx = ldx;
    p.xs = xs;
    p.y = out;
    p.type = type;
    p.ldy = ldo;
    p.n_q_heads = heads->n_heads;
    p.n_kv_heads = heads->n_kv_heads;
    p.head_dim = heads->head_dim;
    p.n_pos = heads->n_pos;
    p.pos = heads->pos;
    p.cos = heads->cos;
    p.sin = heads->sin;
    p.q_norm = heads->q_norm;
    p.k_norm = heads->k_norm;
    p.eps = heads->eps;
    p.err = err;
    return run(kI8Heads, p, {heads->cos, heads->sin, heads->q_norm, heads->k_norm},
               static_cast<cudaStream_t>(stream));
}

}  // extern "C"
