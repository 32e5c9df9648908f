"""The 8-bit integer projections against 64-bit definitions (int8_ref.py):
codes exactly, results within counted roundings."""

import numpy as np
import pytest
import torch

import int8_ref as ref
from ffwd_b200 import native

pytestmark = pytest.mark.gpu

DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def pad16(n):
    return (n + 15) // 16 * 16


def rows(M, K, seed, ld=None):
    """Random codes [M, K] in a buffer whose padding holds other values, and scales."""
    g = gen(seed)
    buf = torch.randint(-127, 128, (M, ld or pad16(K)), device=DEV, generator=g, dtype=torch.int8)
    s = torch.rand(M, device=DEV, generator=g) * 0.02 + 1e-3
    return buf, s


def mat(w, t, K, bias=None):
    return native.i8_mat(w.data_ptr(), t.data_ptr(), w.shape[0], K, w.stride(0),
                         bias.data_ptr() if bias is not None else None)


def within(got, want, bound):
    err = (got.double() - want).abs()
    # Past the type's largest value plus half a step, rounding gives infinity.
    info = torch.finfo(got.dtype)
    over = torch.isinf(got) & (want * got.sign() + bound >= info.max * (1 + info.eps / 4))
    bad = ~((err <= bound) | over)
    assert not bad.any(), (int(bad.sum()), float((err / bound).nan_to_num(1e9).max()),
                           bad.nonzero()[:4].tolist())


def quantise(x, norm=None, eps=1e-6, ldq=None, stream=0):
    M, K = x.shape
    q = torch.full((M, ldq or pad16(K)), 99, dtype=torch.int8, device=DEV)
    s = torch.full((M,), -1.0, device=DEV)
    native.quantize_i8(x.data_ptr(), {v: k for k, v in ref.TYPES.items()}[x.dtype], x.stride(0),
                       q.data_ptr(), q.stride(0), s.data_ptr(), M, K,
                       norm_ptr=norm.data_ptr() if norm is not None else None, eps=eps,
                       stream=stream)
    return q, s


# ---------------------------------------------------------------- rows to codes

# Every width class (1, 4, 16 warps a row; streamed), few and many rows, ragged tails.
QSHAPES = [(1, 1), (3, 7), (1, 256), (5, 257), (400, 384), (1, 1000), (700, 1024), (2, 2048),
           (600, 1537), (301, 4096), (1, 4096), (2, 12288), (310, 5000), (3, 16384), (2, 16385),
           (1, 70001)]


@pytest.mark.parametrize("M,K", QSHAPES)
@pytest.mark.parametrize("dtype", list(ref.TYPES))
@pytest.mark.parametrize("normed", [False, True])
def test_quantise(M, K, dtype, normed):
    g = gen(M * 131 + K)
    x = torch.randn(M, K, device=DEV, generator=g)
    x[:, ::97] *= 8.0
    x = x.to(ref.TYPES[dtype])
    norm = 1.0 + 0.2 * torch.randn(K, device=DEV, generator=g) if normed else None
    q, s = quantise(x, norm)
    qe, se = ref.quantise(x, norm, 1e-6)
    assert torch.equal(q[:, :K], qe)
    assert (q[:, K:] == 99).all()  # padding left alone
    # One rounding; with the norm also the sum of squares: at most 32 terms a
    # thread (K / 512 where the row is streamed) and 9 levels of sums, halved
    # by the root.
    n = 1 if not normed else 2 + (max(32, K // 512 + 8) + 16 + 9) / 2
    assert ((s.double() - se).abs() <= n * ref.U * se).all()


@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_quantise_strided_rows(dtype):
    """Row strides and bases off the vector alignment, and a wide output stride."""
    g = gen(5)
    big = torch.randn(37, 523, device=DEV, generator=g).to(ref.TYPES[dtype])
    x = big[:, 3:500]
    q, s = quantise(x, ldq=1024)
    qe, se = ref.quantise(x)
    assert torch.equal(q[:, :497], qe) and (q[:, 497:] == 99).all()


def test_quantise_codes_next_to_a_border():
    """Values within a few 2^-24 of the border of two codes fall as the exact
    quotient does."""
    K = 1024
    g = gen(7)
    amax = torch.rand(64, 1, device=DEV, generator=g) + 1.0
    k = torch.randint(-126, 126, (64, K), device=DEV, generator=g)
    x = ((k.double() + 0.5) * amax.double() / 127.0).float()
    x = torch.nextafter(x, torch.where(torch.rand(64, K, device=DEV, generator=g) < 0.5,
                                       torch.inf, -torch.inf).float())
    x[:, :1] = amax
    norm = 1.0 + 0.3 * torch.rand(K, device=DEV, generator=g)
    q, _ = quantise(x)
    assert torch.equal(q[:, :K], ref.quantise(x)[0])
    y = (x.double() / norm.double()).float()
    q, _ = quantise(y, norm)
    assert torch.equal(q[:, :K], ref.quantise(y, norm, 1e-6)[0])


@pytest.mark.parametrize("K", [100, 700, 3000, 20000])
@pytest.mark.parametrize("normed", [False, True])
def test_quantise_special_rows(K, normed):
    """Zeros, tiny values, infinities and NaN; the rows beside them keep theirs."""
    g = gen(K)
    x = torch.randn(8, K, device=DEV, generator=g)
    x[1] = 0.0
    x[2, K // 2] = float("inf")
    x[3, K - 1] = float("nan")
    x[4] *= 1e-34
    x[5, 0] = -float("inf")
    norm = 1.0 + 0.2 * torch.randn(K, device=DEV, generator=g) if normed else None
    q, s = quantise(x, norm)
    q = q[:, :K]
    for r in (2, 3, 5):
        assert torch.isnan(s[r]) and (q[r] == 0).all()
    assert s[1] == 0 and (q[1] == 0).all()
    keep = [0, 4, 6, 7]
    qe, se = ref.quantise(x[keep], norm, 1e-6)
    assert torch.equal(q[keep], qe)
    assert ((s[keep].double() - se).abs() <= 60 * ref.U * se + 2.0 ** -149).all()


# ---------------------------------------------------------------- products

# Streaming kernel (up to 4 rows), tiles with K split over a cluster (up to 64
# rows, more for long K) and 256-row tiles; lengths on both sides of a tile, a
# stage and a 16-byte chunk.
SHAPES = [(1, 64, 16), (1, 1024, 2048), (2, 1, 1), (3, 37, 45), (4, 5000, 4500), (8, 5000, 530),
          (8, 10000, 64), (9, 32, 128), (9, 31, 129), (17, 129, 1000), (33, 70, 5000),
          (64, 300, 77), (100, 200, 4200), (65, 33, 130), (128, 257, 1024), (129, 256, 513),
          (20, 40, 3), (300, 40, 1), (300, 1, 20), (200, 300, 8300), (300, 1003, 771), (257, 4096, 384), (1025, 640, 2100)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_gemm(M, N, K, dtype):
    x, s = rows(M, K, M + K)
    w, t = rows(N, K, N + 1)
    b = torch.randn(N, device=DEV, generator=gen(3))
    for bias, kind in ((None, "none"), (b, "gelu"), (b, "silu"), (None, "gelu_tanh")):
        y = torch.full((M, N), float("nan"), dtype=ref.TYPES[dtype], device=DEV)
        native.gemm_i8(mat(w, t, K, bias), x.data_ptr(), x.stride(0), s.data_ptr(), M,
                       y.data_ptr(), dtype, N, act=kind)
        within(y, *ref.gemm(x[:, :K], s, w[:, :K], t, bias, kind, dtype))


def test_gemm_sums_are_exact():
    """The largest sums (every product 127^2, K = 131071) and cancelling ones."""
    K, N = 131071, 48
    for M in (2, 10, 300):
        x = torch.full((M, K + 1), 127, dtype=torch.int8, device=DEV)
        w = torch.full((N, K + 1), 127, dtype=torch.int8, device=DEV)
        w[1, :K] = -128
        w[2, 1:K:2] = -127
        one = torch.ones(max(M, N), device=DEV)
        y = torch.zeros(M, N, device=DEV)
        native.gemm_i8(mat(w, one, K), x.data_ptr(), K + 1, one.data_ptr(), M, y.data_ptr(),
                       "f32", N)
        want = (x[:, :K].double() @ w[:, :K].double().T).float()  # the sum's only rounding
        assert torch.equal(y, want)


@pytest.mark.parametrize("M", [3, 30, 200])
@pytest.mark.parametrize("dtype,N,ld,off", [("f32", 130, 131, 1), ("bf16", 130, 139, 3),
                                            ("f16", 96, 104, 0), ("bf16", 96, 100, 8)])
def test_gemm_output_strides(M, dtype, N, ld, off):
    """Output bases and strides with and without 16-byte alignment; what lies
    around the result is left alone."""
    K = 200
    x, s = rows(M, K, 1)
    w, t = rows(N, K, 2)
    buf = torch.full(((M + 2) * ld + off,), 7.0, dtype=ref.TYPES[dtype], device=DEV)
    native.gemm_i8(mat(w, t, K), x.data_ptr(), x.stride(0), s.data_ptr(), M,
                   buf.data_ptr() + (off + ld) * buf.element_size(), dtype, ld)
    out = buf[off:].view(M + 2, ld)
    within(out[1:M + 1, :N], *ref.gemm(x[:, :K], s, w[:, :K], t, None, "none", dtype))
    assert (out[0] == 7).all() and (out[M + 1] == 7).all() and (out[:, N:] == 7).all()
    assert (buf[:off] == 7).all()


@pytest.mark.parametrize("M,ld", [(4, 96), (4, 97), (40, 97), (333, 96), (333, 97)])
def test_gemm_accumulates(M, ld):
    N, K = 96, 300
    x, s = rows(M, K, 4)
    w, t = rows(N, K, 5)
    y = torch.randn(M, ld, device=DEV, generator=gen(6))
    before = y.clone()
    native.gemm_i8(mat(w, t, K), x.data_ptr(), x.stride(0), s.data_ptr(), M, y.data_ptr(), "f32",
                   ld, accumulate=True)
    want, bound = ref.product(x[:, :K], s, w[:, :K], t)
    want = want + before[:, :N].double()
    within(y[:, :N], want, bound + ref.U * want.abs() + ref.U * bound)
    assert torch.equal(y[:, N:], before[:, N:])


def test_scales_that_are_not_finite_reach_their_row_only():
    M, N, K = 40, 70, 90
    for m in (4, M, 5 * M):
        x, s = rows(m, K, 8)
        w, t = rows(N, K, 9)
        s[1] = float("nan")
        x[1] = 0
        y = torch.zeros(m, N, device=DEV)
        native.gemm_i8(mat(w, t, K), x.data_ptr(), x.stride(0), s.data_ptr(), m, y.data_ptr(),
                       "f32", N)
        assert torch.isnan(y[1]).all()
        keep = [i for i in range(m) if i != 1]
        want, bound = ref.gemm(x[keep][:, :K], s[keep], w[:, :K], t, None, "none", "f32")
        within(y[keep], want, bound)


@pytest.mark.parametrize("M", [2, 20, 300])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_activations_far_out(M, kind):
    """Arguments up to the ends of f32, infinities and NaN (through the bias):
    x far to the right, a zero far to the left, +inf kept, NaN kept."""
    K = 32
    far = [1e5, 3e18, 1e20, 1e30, 3e38, float("inf")]
    bias = torch.tensor(far + [-v for v in far[:-1]] + [float("nan"), 0.0, 6.0, -6.0, 12.0, -12.0],
                        device=DEV)
    N = bias.numel()
    x = torch.zeros(M, K, dtype=torch.int8, device=DEV)
    w = torch.zeros(N, K, dtype=torch.int8, device=DEV)
    one = torch.ones(max(M, N), device=DEV)
    y = torch.zeros(M, N, device=DEV)
    native.gemm_i8(mat(w, one, K, bias), x.data_ptr(), K, one.data_ptr(), M, y.data_ptr(), "f32",
                   N, act=kind)
    n = len(far)
    assert torch.equal(y[:, :n], bias[:n].expand(M, n))
    assert (y[:, n:2 * n - 1] == 0).all()
    assert torch.isnan(y[:, 2 * n - 1]).all()
    near = bias[2 * n:]
    want, bound = ref.act(near.double(), torch.zeros_like(near.double()), kind, "f32")
    within(y[:, 2 * n:], want.expand(M, -1), bound.expand(M, -1) + 2.0 ** -60)


@pytest.mark.parametrize("M,N,K", [(1, 1024, 512), (2, 33, 100), (7, 7000, 48), (24, 2048, 1024),
                                   (129, 127, 130), (700, 1111, 1000), (256, 128, 64),
                                   (4, 300, 2000), (50, 130, 4100), (90, 257, 4100)])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_gated(M, N, K, dtype):
    x, s = rows(M, K, M)
    wg, tg = rows(N, K, 1)
    wu, tu = rows(N, K, 2, ld=pad16(K) + 32)
    b = torch.randn(N, device=DEV, generator=gen(3))
    for kind, bg, bu in (("silu", None, None), ("gelu", b, None), ("gelu_tanh", None, b)):
        h = torch.full((M, N), float("nan"), dtype=ref.TYPES[dtype], device=DEV)
        native.gated_i8(mat(wg, tg, K, bg), mat(wu, tu, K, bu), x.data_ptr(), x.stride(0),
                        s.data_ptr(), M, h.data_ptr(), dtype, N, act=kind)
        within(h, *ref.gated(x[:, :K], s, wg[:, :K], tg, bg, wu[:, :K], tu, bu, kind, dtype))


def tables(n_pos, hd):
    ang = np.outer(np.arange(n_pos), 1e6 ** (-np.arange(hd // 2) / (hd / 2)))
    return (torch.tensor(np.cos(ang), dtype=torch.float32, device=DEV),
            torch.tensor(np.sin(ang), dtype=torch.float32, device=DEV))


def run_qkv(M, K, h, kv, hd, dtype, bias, qn, kn, pos, cos, sin, w, t, x, s, ld=None, err=None):
    N = (h + 2 * kv) * hd
    out = torch.full((M, ld or N), float("nan"), dtype=ref.TYPES[dtype], device=DEV)
    ptr = lambda v: v.data_ptr() if v is not None else None
    hs = native.i8_heads(h, kv, hd, pos.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                         ptr(qn), ptr(kn), 1e-6)
    native.qkv_i8(mat(w, t, K, bias), hs, x.data_ptr(), x.stride(0), s.data_ptr(), M,
                  out.data_ptr(), dtype, ld or N, err_ptr=ptr(err))
    return out


@pytest.mark.parametrize("M,K,h,kv,hd", [(1, 256, 2, 1, 128), (7, 1024, 16, 8, 128),
                                         (5, 100, 7, 1, 64), (9, 130, 1, 1, 64),
                                         (130, 384, 3, 3, 128), (600, 904, 14, 2, 64),
                                         (257, 512, 8, 1, 128), (3, 4096, 2, 1, 64),
                                         (16, 2100, 1, 1, 128), (33, 700, 3, 1, 64),
                                         (64, 1024, 16, 8, 128)])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_qkv(M, K, h, kv, hd, dtype):
    N = (h + 2 * kv) * hd
    x, s = rows(M, K, M)
    w, t = rows(N, K, 11)
    g = gen(12)
    cos, sin = tables(50, hd)
    pos = torch.randint(0, 50, (M,), device=DEV, generator=g, dtype=torch.int32)
    b = torch.randn(N, device=DEV, generator=g)
    qn = 1.0 + 0.2 * torch.randn(hd, device=DEV, generator=g)
    kn = 1.0 + 0.2 * torch.randn(hd, device=DEV, generator=g)
    for bias, a, c in ((None, qn, kn), (b, None, None), (b, None, kn)):
        out = run_qkv(M, K, h, kv, hd, dtype, bias, a, c, pos, cos, sin, w, t, x, s)
        within(out, *ref.qkv(x[:, :K], s, w[:, :K], t, bias, h, kv, hd, pos, cos, sin, a, c,
                             1e-6, dtype))


@pytest.mark.parametrize("M,K,h,kv,hd", [(2400, 2064, 4, 1, 128), (2400, 2048, 4, 1, 128),
                                         (2100, 2300, 7, 2, 64), (5000, 160, 2, 2, 128),
                                         (65, 2048, 8, 2, 128), (127, 4100, 3, 1, 64),
                                         (128, 9000, 1, 1, 128)])
def test_qkv_over_many_tiles(M, K, h, kv, hd):
    """More than one group of row blocks, the last of them short, on both sides of
    the K where the order of the tiles changes; two row blocks of a split K."""
    N = (h + 2 * kv) * hd
    x, s = rows(M, K, 3)
    w, t = rows(N, K, 4)
    cos, sin = tables(M, hd)
    pos = torch.randperm(M, device=DEV, generator=gen(5)).int()
    qn = 1.0 + 0.2 * torch.randn(hd, device=DEV, generator=gen(6))
    out = run_qkv(M, K, h, kv, hd, "bf16", None, qn, None, pos, cos, sin, w, t, x, s)
    within(out, *ref.qkv(x[:, :K], s, w[:, :K], t, None, h, kv, hd, pos, cos, sin, qn, None, 1e-6,
                         "bf16"))


@pytest.mark.parametrize("M,N,K", [(2300, 2600, 5000), (9000, 1600, 8300), (8600, 6200, 2048)])
def test_gated_of_weights_past_the_cache(M, N, K):
    """Groups of up to 26, 15 and 32 row blocks, the last of them short."""
    x, s = rows(M, K, 7)
    wg, tg = rows(N, K, 8)
    wu, tu = rows(N, K, 9)
    h = torch.full((M, N), float("nan"), dtype=torch.float16, device=DEV)
    native.gated_i8(mat(wg, tg, K), mat(wu, tu, K), x.data_ptr(), x.stride(0), s.data_ptr(), M,
                    h.data_ptr(), "f16", N)
    within(h, *ref.gated(x[:, :K], s, wg[:, :K], tg, None, wu[:, :K], tu, None, "silu", "f16"))


@pytest.mark.parametrize("M,N,K", [(7, 1950, 2600), (33, 2048, 9000), (16, 4250, 1100),
                                   (130, 1100, 8200), (100, 4500, 4200)])
def test_gemm_of_few_rows_and_many_clusters(M, N, K):
    """Numbers of channel tiles on both sides of the clusters that fit at a time."""
    x, s = rows(M, K, 1)
    w, t = rows(N, K, 2)
    y = torch.full((M, N), float("nan"), device=DEV)
    native.gemm_i8(mat(w, t, K), x.data_ptr(), x.stride(0), s.data_ptr(), M, y.data_ptr(), "f32", N)
    within(y, *ref.gemm(x[:, :K], s, w[:, :K], t, None, "none", "f32"))


@pytest.mark.parametrize("M", [5, 40, 150])
def test_qkv_positions_outside_the_tables(M):
    h, kv, hd, K = 2, 1, 64, 96
    N = (h + 2 * kv) * hd
    x, s = rows(M, K, 1)
    w, t = rows(N, K, 2)
    cos, sin = tables(10, hd)
    pos = torch.arange(M, device=DEV, dtype=torch.int32) % 10
    pos[2], pos[4] = -1, 10
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = run_qkv(M, K, h, kv, hd, "f32", None, None, None, pos, cos, sin, w, t, x, s, err=err)
    assert err.item() == 5
    assert torch.isnan(out[[2, 4], :(h + kv) * hd]).all()
    good = [i for i in range(M) if i not in (2, 4)]
    pos[2] = pos[4] = 0
    want, bound = ref.qkv(x[:, :K], s, w[:, :K], t, None, h, kv, hd, pos, cos, sin, None, None,
                          1e-6, "f32")
    within(out[good], want[good], bound[good])
    within(out[[2, 4], (h + kv) * hd:], want[[2, 4], (h + kv) * hd:],
           bound[[2, 4], (h + kv) * hd:])


def test_host_memory_is_refused():
    K = 64
    x, s = rows(4, K, 1)
    w, t = rows(32, K, 2)
    y = torch.zeros(4, 32)
    with pytest.raises(native.FfwdError, match="output is not memory of the current device"):
        native.gemm_i8(mat(w, t, K), x.data_ptr(), K, s.data_ptr(), 4, y.data_ptr(), "f32", 32)
    hs = torch.ones(32)
    with pytest.raises(native.FfwdError, match="weight scales is not memory"):
        native.gemm_i8(mat(w, hs, K), x.data_ptr(), K, s.data_ptr(), 4, x.data_ptr(), "f32", 32)


# ---------------------------------------------------------------- together

class Layer:
    """Feed-forward of a decoder layer in int8: norm + quantise, gated block,
    quantise, down projection added to the residual stream."""

    def __init__(self, M, H, I, seed, dtype="bf16"):
        g = gen(seed)
        self.M, self.H, self.I, self.dtype = M, H, I, dtype
        self.x = torch.randn(M, H, device=DEV, generator=g)
        self.norm = 1.0 + 0.1 * torch.randn(H, device=DEV, generator=g)
        self.wf = [torch.randn(n, k, device=DEV, generator=g) / k ** 0.5
                   for n, k in ((I, H), (I, H), (H, I))]
        self.w = [quantise(w) for w in self.wf]
        self.xq = torch.empty(M, pad16(H), dtype=torch.int8, device=DEV)
        self.hq = torch.empty(M, pad16(I), dtype=torch.int8, device=DEV)
        self.xs, self.hs = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
        self.h = torch.empty(M, I, dtype=ref.TYPES[dtype], device=DEV)
        self.mats = [mat(q, s, w.shape[1]) for (q, s), w in zip(self.w, self.wf)]

    def run(self, stream=0):
        M, H, I = self.M, self.H, self.I
        native.quantize_i8(self.x.data_ptr(), "f32", H, self.xq.data_ptr(), self.xq.stride(0),
                           self.xs.data_ptr(), M, H, norm_ptr=self.norm.data_ptr(), eps=1e-6,
                           stream=stream)
        native.gated_i8(self.mats[0], self.mats[1], self.xq.data_ptr(), self.xq.stride(0),
                        self.xs.data_ptr(), M, self.h.data_ptr(), self.dtype, I, stream=stream)
        native.quantize_i8(self.h.data_ptr(), self.dtype, I, self.hq.data_ptr(),
                           self.hq.stride(0), self.hs.data_ptr(), M, I, stream=stream)
        native.gemm_i8(self.mats[2], self.hq.data_ptr(), self.hq.stride(0), self.hs.data_ptr(), M,
                       self.x.data_ptr(), "f32", H, accumulate=True, stream=stream)

    def want(self, x):
        n = x * self.norm / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)
        g, u = n @ self.wf[0].T, n @ self.wf[1].T
        return (g * torch.sigmoid(g) * u) @ self.wf[2].T


@pytest.mark.parametrize("M,H,I", [(1, 256, 640), (7, 1024, 2000), (300, 520, 1100)])
def test_feed_forward_block(M, H, I):
    """The chain against the unquantised block: rows point the same way."""
    L = Layer(M, H, I, M)
    x0 = L.x.clone()
    L.run()
    got, want = (L.x - x0).double(), L.want(x0).double()
    cos = (got * want).sum(1) / (got.norm(dim=1) * want.norm(dim=1))
    # Codes of roughly Gaussian rows (largest value about 4 rms, so a step is
    # 4 / 127 rms and its rounding 0.009 rms) in both operands of two products:
    # a relative error near 0.03, cosine 1 - 0.03^2 / 2 = 0.9995.
    assert cos.min() > 0.998, cos.min()


@pytest.mark.parametrize("M", [2, 30, 200])
def test_captured_and_replayed(M):
    """Captured into a graph and replayed on new inputs, with an eager call of
    other rows between: bitwise the eager results."""
    L, other = Layer(M, 512, 1000, 1), Layer(M + 3, 512, 1000, 2)
    x0 = L.x.clone()
    L.run()
    want = [L.x.clone()]
    L.run()
    want.append(L.x.clone())
    L.x.copy_(x0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        L.run(stream=torch.cuda.current_stream().cuda_stream)
    for w in want:
        graph.replay()
        other.run(stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(L.x, w)


def test_two_streams_at_once():
    a, b = Layer(300, 512, 1000, 3), Layer(5, 512, 1000, 4)
    want = []
    for L in (a, b):
        x0 = L.x.clone()
        L.run()
        want.append(L.x.clone())
        L.x.copy_(x0)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    a.run(stream=sa.cuda_stream)
    b.run(stream=sb.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a.x, want[0]) and torch.equal(b.x, want[1])


def test_offsets_past_32_bits():
    """An output and rows whose offsets pass 2^31 elements and bytes."""
    K, N, M = 64, 16384, 140000
    x, s = rows(M, K, 1, ld=16000)  # 2.2e9 bytes of rows
    w, t = rows(N, K, 2)
    y = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)  # 2.3e9 elements
    native.gemm_i8(mat(w, t, K), x.data_ptr(), x.stride(0), s.data_ptr(), M, y.data_ptr(), "bf16",
                   N)
    tail = slice(M - 200, M)
    within(y[tail], *ref.gemm(x[tail, :K], s[tail], w[:, :K], t, None, "none", "bf16"))
    del y
    q = torch.zeros(M, 16000, dtype=torch.int8, device=DEV)
    src = torch.randn(M, 16001, dtype=torch.bfloat16, device=DEV, generator=gen(1))[:, :70]
    sc = torch.zeros(M, device=DEV)
    native.quantize_i8(src.data_ptr(), "bf16", src.stride(0), q.data_ptr(), 16000, sc.data_ptr(),
                       M, 70)
    assert torch.equal(q[tail, :70], ref.quantise(src[tail])[0])
