"""The 8-bit integer projections, as cases to be timed and compared.

Every case starts from the rows a program holds (bf16 / f16 / f32 activations)
and 8-bit weights with one scale per output channel, and ends with the
projection's result:

* ``linear``: rows quantised to int8 with one scale each, the integer product,
  scales, bias and activation;
* ``gated``: the residual stream's rows RMS-normalised and quantised, gate and
  up projections, activation and product;
* ``qkv``: the same rows into the fused query / key / value projection, each
  query and key head RMS-normalised (where the model does) and rotated to its
  position.

``run`` computes them with elementary torch operations in 32 bits, or, where
``own`` is set, with the framework's operators.
"""

import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _pad16(n):
    return (n + 15) // 16 * 16


def listed():
    return [
        # One token's output projection of a 1024-wide decoder: latency counts.
        dict(name="linear_token", op="linear", M=1, N=1024, K=2048, dtype="bf16", act="none",
             bias=False),
        # A ragged projection: nothing is a multiple of a tile, 32-bit rows.
        dict(name="linear_ragged", op="linear", M=333, N=1003, K=771, dtype="f32", act="none",
             bias=True),
        # Encoder feed-forward expansion, a batch of passages.
        dict(name="linear_gelu", op="linear", M=8192, N=4096, K=1024, dtype="f16", act="gelu",
             bias=True),
        # Down projection of an 8192-token document in a 4096-wide decoder.
        dict(name="linear_down", op="linear", M=8192, N=4096, K=12288, dtype="bf16", act="none",
             bias=False),
        # One token through a gated feed-forward.
        dict(name="gated_token", op="gated", M=1, N=4096, K=1024, dtype="bf16", act="silu"),
        # A short query through a wide gated feed-forward.
        dict(name="gated_query", op="gated", M=24, N=8192, K=2048, dtype="bf16", act="silu"),
        # Ragged, GELU gate.
        dict(name="gated_ragged", op="gated", M=1237, N=1111, K=1000, dtype="f32",
             act="gelu_tanh"),
        # An 8192-token document in a 4096-wide decoder.
        dict(name="gated_document", op="gated", M=8192, N=12288, K=4096, dtype="bf16",
             act="silu"),
        # One short query, 16 query and 8 key/value heads.
        dict(name="qkv_query", op="qkv", M=7, K=1024, heads=16, kv_heads=8, head_dim=128,
             norm=True, bias=False, dtype="bf16", longest=7),
        # Ragged batch without head norms, biased projection, 64-wide heads, one key/value head.
        dict(name="qkv_ragged", op="qkv", M=1001, K=904, heads=14, kv_heads=1, head_dim=64,
             norm=False, bias=True, dtype="f16", longest=400),
        # A packed batch of documents.
        dict(name="qkv_batch", op="qkv", M=32768, K=1024, heads=16, kv_heads=8, head_dim=128,
             norm=True, bias=False, dtype="bf16", longest=2048),
        # An 8192-token document in a 4096-wide decoder, 32 query and 8 key/value heads.
        dict(name="qkv_document", op="qkv", M=8192, K=4096, heads=32, kv_heads=8, head_dim=128,
             norm=True, bias=False, dtype="bf16", longest=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "gated", "qkv"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    while True:
        m = _log(rng, 1, 16384)
        k = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            k = max(16, k // 16 * 16)
        if op == "qkv":
            hd = rng.choice([64, 128])
            kv = rng.choice([1, 2, 4, 8])
            heads = kv * rng.choice([1, 2, 4, 7])
            n = (heads + 2 * kv) * hd
            case = dict(op=op, M=m, K=k, heads=heads, kv_heads=kv, head_dim=hd,
                        norm=rng.random() < 0.5, bias=rng.random() < 0.5, dtype=dtype,
                        longest=_log(rng, 1, 8192))
        else:
            n = _log(rng, 64, 12288)
            if rng.random() < 0.6:
                n = max(8, n // 8 * 8)
            case = dict(op=op, M=m, N=n, K=k, dtype=dtype,
                        act=rng.choice(["silu", "gelu", "gelu_tanh"] +
                                       (["none"] if op == "linear" else [])))
            if op == "linear":
                case["bias"] = rng.random() < 0.5
        if m * n * k * (2 if op == "gated" else 1) <= 1 << 38:
            return case


def _weight(n, k, gen):
    """Random [n, k] weights as int8 rows (stride a multiple of 16 bytes) with a
    scale per row."""
    ld = _pad16(k)
    w = torch.randn(n, k, device="cuda", generator=gen) / math.sqrt(k)
    amax = w.abs().amax(dim=1, keepdim=True)
    q = torch.zeros(n, ld, dtype=torch.int8, device="cuda")
    q[:, :k] = (w * (127.0 / amax)).round().to(torch.int8)
    return q, (amax / 127.0).squeeze(1).contiguous()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k, dt = case["M"], case["K"], _DT[case["dtype"]]
    st = dict(case=case, m=m, k=k, dt=dt)
    # Activations: unit rows with a few large channels, as residual streams have.
    x = torch.randn(m, k, device="cuda", generator=gen)
    x[:, torch.randint(0, k, (max(1, k // 256),), device="cuda", generator=gen)] *= 6.0
    if case["op"] == "linear":
        st["x"] = x.to(dt)
        n = case["N"]
        st["w"], st["ws"] = _weight(n, k, gen)
        st["bias"] = torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
    else:
        st["x"] = x
        st["norm_w"] = 1.0 + 0.1 * torch.randn(k, device="cuda", generator=gen)
    if case["op"] == "gated":
        n = case["N"]
        st["wg"], st["gs"] = _weight(n, k, gen)
        st["wu"], st["us"] = _weight(n, k, gen)
    if case["op"] == "qkv":
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        n = (h + 2 * kv) * hd
        st["w"], st["ws"] = _weight(n, k, gen)
        st["bias"] = torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
        st["qn"] = st["kn"] = None
        if case["norm"]:
            st["qn"] = 1.0 + 0.1 * torch.randn(hd, device="cuda", generator=gen)
            st["kn"] = 1.0 + 0.1 * torch.randn(hd, device="cuda", generator=gen)
        # Packed sequences of random lengths; the position restarts with each.
        rng = np.random.default_rng(seed)
        pos = []
        while len(pos) < m:
            pos.extend(range(int(rng.integers(1, case["longest"] + 1))))
        st["pos"] = torch.tensor(pos[:m], dtype=torch.int32, device="cuda")
        ang = np.outer(np.arange(case["longest"]), 1e6 ** (-np.arange(hd // 2) / (hd / 2)))
        st["cos"] = torch.tensor(np.cos(ang), dtype=torch.float32, device="cuda")
        st["sin"] = torch.tensor(np.sin(ang), dtype=torch.float32, device="cuda")
    st["n"] = n
    st["eps"] = 1e-6
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _plan(st)
    return st


# ---------------------------------------------------------------- the framework's operators

def _plan(st):
    """What a program keeps between calls: the weight descriptors and its buffers."""
    from ffwd_b200 import native

    case, m, k, n, dt = st["case"], st["m"], st["k"], st["n"], st["dt"]

    def mat(q, s, bias):
        return native.i8_mat(q.data_ptr(), s.data_ptr(), n, k, q.stride(0),
                             bias_ptr=bias.data_ptr() if bias is not None else None)

    st["xq"] = torch.empty(m, _pad16(k), dtype=torch.int8, device="cuda")
    st["xs"] = torch.empty(m, dtype=torch.float32, device="cuda")
    st["out"] = torch.empty(m, n, dtype=dt, device="cuda")
    if case["op"] == "gated":
        st["gate"], st["up"] = mat(st["wg"], st["gs"], None), mat(st["wu"], st["us"], None)
    else:
        st["mat"] = mat(st["w"], st["ws"], st["bias"])
    if case["op"] == "qkv":
        ptr = lambda t: t.data_ptr() if t is not None else None
        st["heads"] = native.i8_heads(
            case["heads"], case["kv_heads"], case["head_dim"], st["pos"].data_ptr(),
            st["cos"].data_ptr(), st["sin"].data_ptr(), st["cos"].shape[0],
            q_norm_ptr=ptr(st["qn"]), k_norm_ptr=ptr(st["kn"]), eps=st["eps"])


def _run_own(st):
    from ffwd_b200 import native

    case, m, k = st["case"], st["m"], st["k"]
    x, xq, xs, out = st["x"], st["xq"], st["xs"], st["out"]
    stream = torch.cuda.current_stream().cuda_stream
    op = case["op"]
    xd = case["dtype"] if op == "linear" else "f32"
    norm = None if op == "linear" else st["norm_w"].data_ptr()
    native.quantize_i8(x.data_ptr(), xd, x.stride(0), xq.data_ptr(), xq.stride(0), xs.data_ptr(),
                       m, k, norm_ptr=norm, eps=st["eps"], stream=stream)
    if op == "linear":
        native.gemm_i8(st["mat"], xq.data_ptr(), xq.stride(0), xs.data_ptr(), m, out.data_ptr(),
                       case["dtype"], out.stride(0), act=case["act"], stream=stream)
    elif op == "gated":
        native.gated_i8(st["gate"], st["up"], xq.data_ptr(), xq.stride(0), xs.data_ptr(), m,
                        out.data_ptr(), case["dtype"], out.stride(0), act=case["act"],
                        stream=stream)
    else:
        native.qkv_i8(st["mat"], st["heads"], xq.data_ptr(), xq.stride(0), xs.data_ptr(), m,
                      out.data_ptr(), case["dtype"], out.stride(0), stream=stream)
    return out


# ---------------------------------------------------------------- plain forms

def _act(v, kind):
    if kind == "silu":
        return v / (1.0 + torch.exp(-v))
    if kind == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _quantised(st):
    # In 64 bits: a value next to the border of two steps falls to either side
    # with the last bits of its quotient.  A tensor divides (a Python number
    # would multiply by its rounded reciprocal): a value on the border then
    # goes to the even code.
    x = st["x"].double()
    if st["case"]["op"] != "linear":
        x = x * st["norm_w"] / torch.sqrt((x * x).mean(dim=1, keepdim=True) + st["eps"])
    amax = x.abs().amax(dim=1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    return (x / scale).round().float(), scale.float()


def _product(q, s, w, ws, k):
    return (q @ w[:, :k].float().T) * s * ws


def _run_plain(st):
    case, m, k = st["case"], st["m"], st["k"]
    q, s = _quantised(st)
    if case["op"] == "gated":
        g = _product(q, s, st["wg"], st["gs"], k)
        u = _product(q, s, st["wu"], st["us"], k)
        return (_act(g, case["act"]) * u).to(st["dt"])
    y = _product(q, s, st["w"], st["ws"], k)
    if st["bias"] is not None:
        y = y + st["bias"]
    if case["op"] == "linear":
        return _act(y, case["act"]).to(st["dt"])
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    y = y.view(m, h + 2 * kv, hd)
    qk, v = y[:, :h + kv], y[:, h + kv:]
    if case["norm"]:
        w = torch.cat([st["qn"].expand(h, hd), st["kn"].expand(kv, hd)])
        qk = qk / torch.sqrt((qk * qk).mean(dim=2, keepdim=True) + st["eps"]) * w
    pos = st["pos"].long()
    c, sn = st["cos"][pos][:, None, :], st["sin"][pos][:, None, :]
    a, b = qk[..., :hd // 2], qk[..., hd // 2:]
    qk = torch.cat([a * c - b * sn, b * c + a * sn], dim=2)
    return torch.cat([qk, v], dim=1).reshape(m, -1).to(st["dt"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    m, k = case["M"], case["K"]
    n = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"] if case["op"] == "qkv" \
        else case["N"]
    mats = 2 if case["op"] == "gated" else 1
    esz = 4 if case["dtype"] == "f32" else 2
    xsz = esz if case["op"] == "linear" else 4
    nbytes = m * k * xsz + mats * n * (k + 4) + m * n * esz
    if case["op"] != "linear":
        nbytes += 4 * k
    if case.get("bias"):
        nbytes += 4 * n
    if case["op"] == "qkv":
        nbytes += 4 * m + 4 * case["longest"] * case["head_dim"]
        if case["norm"]:
            nbytes += 8 * case["head_dim"]
    return {"bytes": nbytes, "flops": 2 * m * n * k * mats}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    st = _inputs(case, seed)
    d = torch.float64
    x = st["x"].to(d)
    if "norm_w" in st:
        rms = torch.linalg.vector_norm(x, dim=1) / math.sqrt(case["K"])
        x = st["norm_w"].to(d) * (x / torch.sqrt(rms ** 2 + st["eps"])[:, None])
    largest = x.abs().max(dim=1).values
    step = torch.true_divide(largest, torch.tensor(127.0, dtype=d, device=largest.device))
    codes = torch.round(x / step[:, None])

    def proj(w, scale):
        ints = torch.einsum("mk,nk->mn", codes, w[:, :case["K"]].to(d))
        return ints * torch.outer(step, scale.to(d))

    def act(v):
        if case["act"] == "silu":
            return v * torch.special.expit(v)
        if case["act"] == "gelu":
            return v * torch.special.ndtr(v)
        if case["act"] == "gelu_tanh":
            return v * torch.special.expit(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
        return v

    if case["op"] == "gated":
        return act(proj(st["wg"], st["gs"])) * proj(st["wu"], st["us"])
    y = proj(st["w"], st["ws"])
    if case["bias"]:
        y += st["bias"].to(d)
    if case["op"] == "linear":
        return act(y)
    hd, half = case["head_dim"], case["head_dim"] // 2
    rot = torch.complex(st["cos"].to(d), st["sin"].to(d))[st["pos"].long()]
    for head in range(case["heads"] + case["kv_heads"]):
        col = y[:, head * hd:(head + 1) * hd]
        if case["norm"]:
            w = st["qn"] if head < case["heads"] else st["kn"]
            col *= w.to(d) / torch.sqrt(torch.mean(col ** 2, dim=1, keepdim=True) + st["eps"])
        z = torch.complex(col[:, :half], col[:, half:]) * rot
        y[:, head * hd:(head + 1) * hd] = torch.cat([z.real, z.imag], dim=1)
    return y
