"""Models with their projections in 8-bit integers (ffwd_b200_set_linear_i8)
against a numpy model that quantises the same way, and against the reference's
golden embeddings.

Gates.  Against the numpy model the differences are the 16-bit plan's (its
roundings of qkv, attention output and FFN activation, and the codes they
move): that plan's cosine gate, 0.999.  Against the unquantised reference: a
code is off by at most half a step, 1 / sqrt(12) of one in the mean square; a
row whose largest value is 4 (Gaussian) to 10 (gated activations) times its rms
is then off by 0.009 to 0.023 of itself, a product of two such operands by up
to 0.03, and eight products in two layers by up to 0.03 sqrt(8) = 0.09: cosine
1 - 0.09^2 / 2 = 0.996; the gate is 0.99."""

import numpy as np
import pytest
import torch

from ffwd_b200 import native
from golden_util import load
from helpers import cos_rows
from oracle import forward as of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _restore_defaults():
    yield
    L = native.lib()
    L.ffwd_b200_set_weights_default()
    L.ffwd_b200_set_fast_gemm(b"f32")
    L.ffwd_b200_set_linear_i8(0)


def codes(v):
    s = np.abs(v).max(1, keepdims=True).astype(np.float64) / 127.0
    return np.rint(v / np.where(s > 0, s, 1.0)), s


class I8Weight:
    """Stands for a projection's weights in `x @ w.T`: both sides quantised."""

    __array_ufunc__ = None

    def __init__(self, w):
        self.q, self.s = codes(w)

    @property
    def T(self):
        return self

    def __rmatmul__(self, x):
        q, s = codes(x)
        return ((q @ self.q.T) * s * self.s.T).astype(np.float32)


def i8_oracle(d):
    m = of.OracleModel(d)
    for name in list(m.t):
        if name.endswith("proj.weight") or ".dense.weight" in name or \
                ".self.query.weight" in name or ".self.key.weight" in name or \
                ".self.value.weight" in name:
            m.t[name] = I8Weight(m.t[name])
    return m


CASES = [
    # fixture, gemm mode, weight storage
    ("qwen3_last", "bf16", "file"),
    ("qwen3_edges", "bf16", "file"),
    ("qwen3_bidir", "bf16", "file"),
    ("qwen2_mean", "bf16", "file"),  # projection biases, no head norms
    ("qwen3_f16", "f32", "f16"),     # f16 attention
    ("minilm_f32", "bf16", "file"),  # head_dim 32 encoder
    ("bge_bf16_cls", "bf16", "file"),
    ("xlmr_mean", "16f", "file"),
    ("bert_tanh_cls", "bf16", "file"),
]


@pytest.mark.parametrize("name,mode,wdt", CASES)
def test_model(name, mode, wdt, model_root):
    spec, d, seqs, expected = load(name, model_root)
    m = native.B200Model(d, gemm_mode=mode, weight_dtype=wdt, linear_i8=True)
    try:
        assert m.precision == 5
        out = m.encode_batch(seqs)
        again = m.encode_batch(seqs)
    finally:
        m.close()
    assert np.isfinite(out).all()
    assert np.array_equal(out, again)
    cos = cos_rows(out, i8_oracle(d).encode_batch(seqs))
    assert cos.min() >= 0.999, cos.min()
    cos = cos_rows(out, expected)
    assert cos.min() >= 0.99, cos.min()


@pytest.mark.parametrize("name", ["qwen3_last", "minilm_f32"])
def test_short_inputs(name, model_root):
    """Batches of up to 8 tokens (the kernels for few rows), and their rows among
    longer sequences."""
    spec, d, seqs, _ = load(name, model_root)
    short = [np.asarray(s)[:n] for s, n in zip(seqs, (1, 3, 8, 5))]
    m = native.B200Model(d, gemm_mode="bf16", weight_dtype="file", linear_i8=True)
    try:
        alone = np.concatenate([m.encode_batch([s]) for s in short])
        mixed = m.encode_batch(short + [seqs[0]])[:len(short)]
    finally:
        m.close()
    ref = i8_oracle(d).encode_batch(short)
    assert cos_rows(alone, ref).min() >= 0.999
    assert cos_rows(mixed, ref).min() >= 0.999


def test_device_and_no_allocation_entries(model_root):
    """The device-resident entry and the no-allocation one, bit for bit."""
    spec, d, seqs, _ = load("qwen3_last", model_root)
    seqs = [np.asarray(s)[:60] for s in seqs[:4]]
    m = native.B200Model(d, gemm_mode="bf16", weight_dtype="file", linear_i8=True)
    try:
        ids = torch.tensor(np.concatenate(seqs), dtype=torch.int32, device="cuda")
        offs = np.concatenate([[0], np.cumsum([len(s) for s in seqs])])
        a = torch.zeros(len(seqs), m.hidden, device="cuda")
        b = torch.ones(len(seqs), m.hidden, device="cuda")
        m.encode_device(ids.data_ptr(), offs, a.data_ptr())
        assert m.encode_device_noalloc(ids.data_ptr(), offs, b.data_ptr()) == 0
        assert torch.equal(a, b)
        assert np.array_equal(a.cpu().numpy(), m.encode_batch(seqs))
    finally:
        m.close()


def test_the_plan_is_chosen_per_load(model_root):
    """An 8-bit model and a 16-bit one side by side; the switch is the load's."""
    spec, d, seqs, expected = load("qwen3_last", model_root)
    a = native.B200Model(d, gemm_mode="bf16", weight_dtype="file", linear_i8=True)
    b = native.B200Model(d, gemm_mode="bf16", weight_dtype="file")
    try:
        assert (a.precision, b.precision) == (5, 0)
        x, y = a.encode_batch(seqs), b.encode_batch(seqs)
        assert cos_rows(y, expected).min() >= 0.999
        assert not np.array_equal(x, y)
        assert np.array_equal(x, a.encode_batch(seqs))
    finally:
        a.close()
        b.close()


def test_late_interaction_and_spans(model_root):
    """Token vectors and span means of 8-bit models."""
    from golden_util import load_spans
    from helpers import small_spec
    from ffwd_b200 import synth

    L = native.lib()
    d = synth.ensure_model(small_spec("qwen3-late-2l"), model_root)
    ids = np.arange(100, 140, dtype=np.int32)
    L.ffwd_b200_set_linear_i8(1)
    late = native.B200Late(d, gemm_mode="bf16")
    L.ffwd_b200_set_linear_i8(0)
    try:
        vec = late.encode_tokens(ids)
    finally:
        late.close()
    assert cos_rows(vec, of.OracleLate(d).encode_tokens(ids)).min() >= 0.99
    spec, d, docs, spans, expected = load_spans("qwen3_spans", model_root)
    m = native.B200Model(d, gemm_mode="bf16", weight_dtype="file", linear_i8=True)
    try:
        got = m.encode_spans_batch(docs, spans)
    finally:
        m.close()
    assert cos_rows(got, expected).min() >= 0.99


def test_exact_plans_are_refused(model_root):
    spec, d, seqs, _ = load("minilm_f32", model_root)
    for mode in ("f32", "tf32"):
        with pytest.raises(native.FfwdError, match="16-bit plan"):
            native.B200Model(d, gemm_mode=mode, weight_dtype="file", linear_i8=True)
