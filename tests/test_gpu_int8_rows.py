"""Rows whose products with the norm's weights leave f32's normal range, against
the 64-bit definition (int8_ref.quantise): codes exactly, scales to a rounding."""

import pytest
import torch

import int8_ref as ref
from test_gpu_int8 import DEV, gen, quantise

pytestmark = pytest.mark.gpu

# Each width class: one to 16 warps a row, by element, streamed; few and many rows.
WIDTHS = [(9, 100), (400, 256), (9, 1000), (400, 700), (400, 3000), (9, 4096), (400, 8192),
          (9, 20000), (400, 771), (9, 16390)]
TINY = [1e-29, 1e-31, 1e-36, 1e-38, 1e-40, 3e-44]


def check(q, s, x, norm, eps, terms):
    """Where the sums are f32's: at most `terms` roundings of squares and sums,
    halved by the root, and four of the quotients; half of f32's smallest step
    where the scale is below its normal range."""
    qe, se = ref.quantise(x, norm, torch.tensor(eps, dtype=torch.float32).item())
    assert torch.equal(q[:, :x.shape[1]], qe)
    assert (q[:, x.shape[1]:] == 99).all()  # padding left alone
    n = 4 + terms / 2
    assert ((s.double() - se).abs() <= n * ref.U * se + 2.0 ** -150).all()


@pytest.mark.parametrize("M,K", WIDTHS)
@pytest.mark.parametrize("eps", [1e-6, 1e-40])
def test_tiny_rows_with_a_norm(M, K, eps):
    """Row r is of size TINY[r % 6] (the last ones a few of f32's smallest steps),
    weights around 1.45: the rounded largest product is then far from the exact
    one.  With eps = 1e-40 the mean of squares itself leaves f32."""
    g = gen(K)
    size = torch.tensor(TINY, device=DEV)[torch.arange(M, device=DEV) % len(TINY)]
    x = (torch.randn(M, K, device=DEV, generator=g).double() * size[:, None].double()).float()
    norm = 1.45 + 0.2 * torch.rand(K, device=DEV, generator=g)
    q, s = quantise(x, norm, eps=eps)
    check(q, s, x, norm, eps, max(32, K // 512 + 8) + 9)


@pytest.mark.parametrize("M,K", WIDTHS)
def test_one_step_times_a_weight(M, K):
    """One of f32's smallest steps times 1.45 rounds back to one step; the codes
    are the exact products' all the same."""
    g = gen(M + K)
    x = torch.zeros(M, K, device=DEV)
    x[:, ::3] = 2.0 ** -149
    x[:, 1::3] = -(2.0 ** -149)
    norm = 0.6 + 0.85 * torch.rand(K, device=DEV, generator=g)
    norm[0] = 1.45
    q, s = quantise(x, norm, eps=1e-6)
    check(q, s, x, norm, 1e-6, 0)


@pytest.mark.parametrize("M,K", WIDTHS)
def test_rows_of_zeros_among_others(M, K):
    """Zero rows, rows that the weights make zero, and whole ones between them."""
    g = gen(K + 1)
    x = torch.randn(M, K, device=DEV, generator=g)
    x[1::3] = 0.0
    norm = 1.0 + 0.2 * torch.randn(K, device=DEV, generator=g)
    norm[K // 2:] = 0.0
    x[2::3, :K // 2] = 0.0
    q, s = quantise(x, norm, eps=1e-6)
    assert (s[1::3] == 0).all() and (s[2::3] == 0).all()
    check(q, s, x, norm, 1e-6, max(32, K // 512 + 8) + 9)
