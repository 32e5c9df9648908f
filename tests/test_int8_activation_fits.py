"""The constants of the 8-bit kernels' activations (int8_epi.cuh), read from the
source and checked in 64 bits: what the GPU test takes as exact."""

import math
import os
import re

import numpy as np
import torch

EPI = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ffwd_b200",
                   "csrc", "int8_epi.cuh")


def constants(name):
    """The f32 constants of `both(...)` in a function, in order."""
    text = open(EPI).read()
    body = text[text.index(f"float2 {name}(float2 x) {{"):]
    body = body[:body.index("\n}\n")]
    out = []
    for expr in re.findall(r"both\(([^()]*)\)", body):
        v = np.float32(1.0)
        for f in expr.split("*"):
            v = np.float32(v * np.float32(f.strip().rstrip("f")))
        out.append(float(v))
    return out


def gelu_erf_fit(x):
    """The kernel's gelu_erf without its roundings."""
    c = constants("gelu_erf")
    assert len(c) == 9  # slope of t, 1, six coefficients, exponent
    t = 1.0 / (c[1] + c[0] * x.abs())
    a = torch.full_like(x, c[2])
    for k in c[3:8]:
        a = a * t + k
    return x.clamp(min=0) - x.abs() * a * t * torch.exp2(c[8] * x * x)


def near(a, b):
    """a is b rounded to f32."""
    return abs(a - b) <= 2.0 ** -24 * abs(b)


def test_gelu_erf():
    """Off by at most 2e-8, and in the tail by little of the result itself."""
    x = torch.linspace(-12, 12, 960001, dtype=torch.float64)
    want = 0.5 * x * torch.special.erfc(-x * math.sqrt(0.5))
    err = (gelu_erf_fit(x) - want).abs()
    assert err.max() <= 2e-8
    for lo, hi, rel in ((-1, 0, 1e-6), (-3, -1, 1e-5), (-5, -3, 3e-5), (-7, -5, 2e-4),
                        (-9, -7, 1e-3), (-12, -9, 2e-3)):
        m = (x >= lo) & (x < hi)
        assert (err[m] <= rel * want[m].abs()).all(), (lo, hi)


def test_silu():
    hi, lo, again, ln2 = (constants("silu")[i] for i in (0, 1, 2, 3))
    assert hi == again and abs(hi + lo + 1 / math.log(2)) < 2.0 ** -48 and near(ln2, math.log(2))


def test_gelu_tanh():
    cubic, linear = constants("gelu_tanh")
    k = -2 / math.log(2) * math.sqrt(2 / math.pi)
    assert near(linear, k) and near(cubic, 0.044715 * k)
