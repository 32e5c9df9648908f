"""The same rows in calls of different numbers of rows, which different kernels
take: byte dot products, tiles of up to 128 rows with K split, 256-row tiles.
Sums are integers and the epilogues round alike, so the results are the same
bits, but for the head norms' sums of squares, which are added in other orders."""

import pytest
import torch

import int8_ref as ref
from ffwd_b200 import native
from test_gpu_int8 import DEV, gen, mat, rows, run_qkv, tables, within

pytestmark = pytest.mark.gpu

COUNTS = [1, 2, 4, 16, 33, 65, 130, 600]


def parts(x, s):
    """The first M rows, for each M."""
    return [(m, x[:m], s[:m]) for m in COUNTS]


@pytest.mark.parametrize("K", [200, 1024, 2500, 8300])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_products(K, dtype):
    N = 300
    x, s = rows(COUNTS[-1], K, 1)
    w, t = rows(N, K, 2)
    u, v = rows(N, K, 3)
    b = torch.randn(N, device=DEV, generator=gen(4))
    for kind in ("none", "silu", "gelu", "gelu_tanh"):
        whole = None
        for M, xm, sm in reversed(parts(x, s)):
            y = torch.full((M, N), float("nan"), dtype=ref.TYPES[dtype], device=DEV)
            h = y.clone()
            native.gemm_i8(mat(w, t, K, b), xm.data_ptr(), x.stride(0), sm.data_ptr(), M,
                           y.data_ptr(), dtype, N, act=kind)
            if kind != "none":
                native.gated_i8(mat(w, t, K, b), mat(u, v, K), xm.data_ptr(), x.stride(0),
                                sm.data_ptr(), M, h.data_ptr(), dtype, N, act=kind)
            if whole is None:
                whole = y, h
            assert torch.equal(y, whole[0][:M]), M
            assert kind == "none" or torch.equal(h, whole[1][:M]), M


@pytest.mark.parametrize("K", [256, 1100, 4200])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_heads(K, hd, dtype):
    h, kv = 3, 1
    N = (h + 2 * kv) * hd
    x, s = rows(COUNTS[-1], K, 5)
    w, t = rows(N, K, 6)
    cos, sin = tables(90, hd)
    pos = torch.randint(0, 90, (COUNTS[-1],), device=DEV, generator=gen(7), dtype=torch.int32)
    b = torch.randn(N, device=DEV, generator=gen(8))
    qn = 1.0 + 0.2 * torch.randn(hd, device=DEV, generator=gen(9))
    # Queries normed, keys and values not.
    want, bound = ref.qkv(x[:, :K], s, w[:, :K], t, b, h, kv, hd, pos, cos, sin, qn, None, 1e-6,
                          dtype)
    whole = None
    for M, xm, sm in reversed(parts(x, s)):
        out = run_qkv(M, K, h, kv, hd, dtype, b, qn, None, pos, cos, sin, w, t, xm, sm)
        if whole is None:
            whole = out
        assert torch.equal(out[:, h * hd:], whole[:M, h * hd:]), M
        within(out[:, :h * hd], want[:M, :h * hd], bound[:M, :h * hd])


@pytest.mark.parametrize("M", [1, 2, 3, 4])
@pytest.mark.parametrize("N", [100, 4737, 9999])
@pytest.mark.parametrize("K", [45, 700])
def test_few_rows_of_every_width(M, N, K):
    """One, two and four weight rows a warp, their last ones past the matrix."""
    x, s = rows(M, K, 1)
    w, t = rows(N, K, 2)
    u, v = rows(N, K, 3)
    y = torch.full((M, N), float("nan"), device=DEV)
    h = y.clone()
    native.gemm_i8(mat(w, t, K), x.data_ptr(), x.stride(0), s.data_ptr(), M, y.data_ptr(), "f32", N)
    native.gated_i8(mat(w, t, K), mat(u, v, K), x.data_ptr(), x.stride(0), s.data_ptr(), M,
                    h.data_ptr(), "f32", N)
    within(y, *ref.gemm(x[:, :K], s, w[:, :K], t, None, "none", "f32"))
    within(h, *ref.gated(x[:, :K], s, w[:, :K], t, None, u[:, :K], v, None, "silu", "f32"))
