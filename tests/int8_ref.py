"""The 8-bit integer projections in 64 bits, with error bounds (test code only).

Bounds count roundings: u = 2^-24 is half a step of f32, `half(t)` half a step
of the output type.
"""

import math

import torch

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def tiny(dtype):
    """Half of the type's smallest step next to zero."""
    return torch.finfo(TYPES[dtype]).smallest_normal * torch.finfo(TYPES[dtype]).eps / 2


def quantise(x, norm=None, eps=0.0):
    """(codes int8, scales f64) of x [M, K]."""
    v = x.double()
    if norm is not None:
        v = v * norm.double()
    amax = v.abs().amax(1)
    s = amax / torch.full_like(amax, 127.0)  # a tensor: a number's reciprocal would be rounded
    q = torch.where(s[:, None] > 0, (v / s[:, None]).round(), torch.zeros_like(v))
    if norm is not None:
        s = s / torch.sqrt((x.double() ** 2).mean(1) + eps)
    return q.to(torch.int8), s


def product(q, s, w, t, bias=None):
    """(y, bound): s x t times the integer sums, plus bias.  The kernel rounds
    the sum to f32, its product with s, and the fused product with t and sum
    with the bias: 2 u of the product and u of the result."""
    a = (q.double() @ w.double().T) * s.double()[:, None] * t.double()
    y = a if bias is None else a + bias.double()
    return y, 2 * U * a.abs() + U * y.abs()


def act(y, bound, kind, dtype):
    """(act(y), bound).  The activations' slopes are below 1.13.

    f32: SiLU's expf (2 ulp = 4 u), sum and quotient: 7 u of the result.  GELU:
    erff / tanhf (2 ulp), their argument (at most 6 u of it, which moves them
    by at most 0.5 of that) and the sum and products: below 9 u of y.
    16-bit: SiLU by __expf (2 + 1.173 |y| ulp) and __fdividef (2 ulp)."""
    if kind == "none":
        return y, bound
    if kind == "silu":
        a = y * torch.sigmoid(y)
        own = 7 * U * a.abs() if dtype == "f32" else (5 + 1.2 * y.abs()) * 2 * U * a.abs()
    elif kind == "gelu":
        a = 0.5 * y * torch.special.erfc(-y * math.sqrt(0.5))
        own = 9 * U * y.abs()
    else:
        a = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        own = 9 * U * y.abs()
    return a, 1.13 * bound + own


def store(y, bound, dtype):
    """(y, bound) after rounding to the output type."""
    return y, bound + half(dtype) * (y.abs() + bound) + tiny(dtype)


def gemm(q, s, w, t, bias, kind, dtype):
    return store(*act(*product(q, s, w, t, bias), kind, dtype), dtype)


def gated(q, s, wg, tg, bg, wu, tu, bu, kind, dtype):
    a, da = act(*product(q, s, wg, tg, bg), kind, dtype)
    u, du = product(q, s, wu, tu, bu)
    return store(a * u, da * u.abs() + a.abs() * du + da * du + U * (a * u).abs(), dtype)


def qkv(q, s, w, t, bias, n_heads, n_kv, hd, pos, cos, sin, qn, kn, eps, dtype):
    y, dy = product(q, s, w, t, bias)
    M = y.shape[0]
    y, dy = y.view(M, -1, hd).clone(), dy.view(M, -1, hd).clone()
    for h in range(n_heads + n_kv):
        wn = qn if h < n_heads else kn
        z, dz = y[:, h], dy[:, h]
        if wn is not None:
            # Sum of hd squares in order (hd u), its root, quotient and two
            # products; the inputs' own errors move the RMS by at most their
            # largest relative size, bounded by their norm over the row's.
            inv = 1.0 / torch.sqrt((z ** 2).mean(1, keepdim=True) + eps)
            rel = (hd / 2 + 6) * U + dz.norm(dim=1, keepdim=True) * inv / math.sqrt(hd)
            wd = wn.double()
            dz = dz * inv * wd.abs() + rel * (z * inv * wd).abs()
            z = z * inv * wd
        c, sn = cos.double()[pos.long()], sin.double()[pos.long()]
        a, b = z[:, :hd // 2], z[:, hd // 2:]
        da, db = dz[:, :hd // 2], dz[:, hd // 2:]
        y[:, h] = torch.cat([a * c - b * sn, b * c + a * sn], 1)
        mag = a.abs() + b.abs()
        dy[:, h] = torch.cat([da + db, da + db], 1) + 3 * U * torch.cat([mag, mag], 1)
    return store(y.reshape(M, -1), dy.reshape(M, -1), dtype)
