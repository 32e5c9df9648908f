"""The 8-bit kernels' activations against 64 bits, within bounds counted from
their own arithmetic (ex2.approx off by at most 2^-22 of the result, rcp.approx by
2^-23, both flushing results below 2^-126): arguments come in through the bias of
codes that are all zero, so they are exact."""

import math

import pytest
import torch

import int8_ref as ref
from ffwd_b200 import native
from test_gpu_int8 import DEV, mat, within
from test_int8_activation_fits import gelu_erf_fit

pytestmark = pytest.mark.gpu

U = ref.U


def exact(x, kind):
    """(activation, bound of the kernel's f32 arithmetic) in 64 bits."""
    if kind == "silu":
        # d = 2^e: 4 u of ex2, 1 of the fused correction (whose own square is below
        # 1e-3 u); 1 + d: 1; its reciprocal: 2; the product: 1.
        y = x * torch.sigmoid(x)
        return y, 9 * U * y.abs() + 2.0 ** -118
    if kind == "gelu_tanh":
        # e: the square, its constant, the fused sum and its constant, the product
        # with x: 4 u of e, which moves 2^e by |e| ln 2 times that; then as above.
        v2 = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        y = x * torch.sigmoid(v2)
        return y, (4 * torch.sigmoid(-v2) * (v2.abs() + 1) + 4) * U * y.abs() + 2.0 ** -118
    # GELU, erf form.  t: 4 u (constant, sum, reciprocal); the polynomial: with S the
    # sum of its terms' magnitudes, 6 u S of its steps, u S of its coefficients, at
    # most 24 u S of t's error (degree 5); then the product with t: 6 u, the power: 4 u and x^2 / 2 times 3 u of its exponent, the products: 2 u, the
    # final sum 1 u of the result.
    y = 0.5 * x * torch.special.erfc(-x * math.sqrt(0.5))
    fit = (gelu_erf_fit(x.cpu()).to(x.device) - y).abs()  # at most 2e-8
    t = 1.0 / (1.0 + 0.4 * x.abs() * math.sqrt(0.5))
    S = torch.zeros_like(x)
    for c in (0.20369884, 0.7232648, 0.3939358, 0.48692873, 0.15432052, 0.23312044):
        S = S * t + 0.5 * c
    part = x.abs() * torch.exp(-x * x / 2) * t * S
    return y, fit + (6 + 1 + 24 + 6 + 4 + 2 + 1.5 * x * x) * U * part + U * y.abs() + 2.0 ** -118


def arguments():
    x = torch.cat([torch.linspace(-12, 12, 4001), torch.linspace(-1e-3, 1e-3, 101),
                   torch.tensor([-1e-30, 1e-30, -3e-39, 20.0, -20.0, -40.0, 60.0, -80.0])])
    return x.to(DEV)


@pytest.mark.parametrize("M", [1, 20, 150])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_sweep(M, dtype, kind):
    x = arguments()
    N, K = x.numel(), 16
    q = torch.zeros(M, K, dtype=torch.int8, device=DEV)
    w = torch.zeros(N, K, dtype=torch.int8, device=DEV)
    one = torch.ones(max(M, N), device=DEV)
    y = torch.full((M, N), float("nan"), dtype=ref.TYPES[dtype], device=DEV)
    native.gemm_i8(mat(w, one, K, x), q.data_ptr(), K, one.data_ptr(), M, y.data_ptr(), dtype, N,
                   act=kind)
    want, bound = ref.store(*exact(x.double(), kind), dtype)
    within(y, want.expand(M, -1), bound.expand(M, -1))


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_bound_is_tight_enough(kind):
    """The f32 bound is below 1 % of every result above 1e-33 (the flushed results'
    2^-118 is 3e-36), so the tails are tested too."""
    y, bound = exact(arguments().double(), kind)
    m = y.abs() > 1e-33
    assert (bound[m] < 0.01 * y[m].abs()).all()
