"""The 8-bit plan on whole models: widths that take each form of the encoders'
LayerNorm with quantisation, the plan's use by late interaction, sequences alone
and among others."""

import numpy as np
import pytest

from ffwd_b200 import native, synth
from golden_util import load
from helpers import cos_rows, small_spec
from oracle import forward as of
from test_gpu_int8_model import I8Weight, _restore_defaults, i8_oracle  # noqa: F401

pytestmark = pytest.mark.gpu

# Hidden sizes: whole groups of 256 columns (256, 512, 768, 1024), ragged ones in two
# groups and in four (128, 384; 640, 896), and past 1024 a LayerNorm and a
# quantisation of their own (1152).
ENCODERS = [(128, 2), (256, 4), (384, 12), (512, 8), (640, 10), (768, 12), (896, 14), (1024, 16),
            (1152, 18)]


@pytest.mark.parametrize("hidden,heads", ENCODERS)
@pytest.mark.parametrize("mode", ["bf16", "16f"])
def test_encoder_widths(hidden, heads, mode, model_root):
    """Against the model that quantises the same way: only the 16-bit plan's
    roundings differ, so its gate."""
    d = synth.ensure_model(synth.spec("bge-base", n_layers=2, hidden=hidden, n_heads=heads,
                                      n_kv_heads=heads, head_dim=hidden // heads,
                                      intermediate=2 * hidden, vocab=1024, pooling="mean"),
                           model_root)
    rng = np.random.default_rng(hidden)
    seqs = [rng.integers(0, 1024, n).astype(np.int32) for n in (1, 5, 40, 131, 300)]
    m = native.B200Model(d, gemm_mode=mode, weight_dtype="file", linear_i8=True)
    try:
        out = m.encode_batch(seqs)
        assert np.array_equal(out, m.encode_batch(seqs))
    finally:
        m.close()
    cos = cos_rows(out, i8_oracle(d).encode_batch(seqs))
    assert cos.min() >= 0.999, cos


def i8_late(d):
    """OracleLate over quantised projections."""
    m = of.OracleLate(d)
    for name in list(m.base.t):
        if name.endswith("proj.weight"):
            m.base.t[name] = I8Weight(m.base.t[name])
    return m


def test_late_interaction_runs_the_plan(model_root):
    """Token vectors differ from the 16-bit plan's, and agree with a model that
    quantises the same way.

    Gate.  A 16-bit rounding next to a border moves a code by a whole step.  Were all
    of them moved, the two models' rounding errors would be independent, each at most
    0.09 of a row after two layers (eight products of two operands that are each off
    by up to 0.023 of themselves: 0.03 sqrt(8)): sqrt(2) 0.09 between them, cosine 1 -
    0.127^2 / 2 = 0.992.  Single tokens, unlike pooled rows, average nothing."""
    d = synth.ensure_model(small_spec("qwen3-late-2l"), model_root)
    ids = np.arange(100, 140, dtype=np.int32)
    vec = {}
    for i8 in (False, True):
        late = native.B200Late(d, gemm_mode="bf16", linear_i8=i8)
        try:
            vec[i8] = late.encode_tokens(ids)
        finally:
            late.close()
    assert not np.array_equal(vec[False], vec[True])
    assert cos_rows(vec[False], of.OracleLate(d).encode_tokens(ids)).min() >= 0.999
    assert cos_rows(vec[True], i8_late(d).encode_tokens(ids)).min() >= 0.992


@pytest.mark.parametrize("name", ["qwen3_last", "qwen2_mean", "minilm_f32", "bge_bf16_cls"])
def test_alone_and_among_others(name, model_root):
    """Another batch changes a row by the 16-bit plan's roundings (attention windows
    of short sequences, head norms) and the codes that these move: its gate."""
    spec, d, seqs, _ = load(name, model_root)
    m = native.B200Model(d, gemm_mode="bf16", weight_dtype="file", linear_i8=True)
    try:
        alone = np.concatenate([m.encode_batch([s]) for s in seqs])
        together = m.encode_batch(seqs)
    finally:
        m.close()
    cos = cos_rows(alone, together)
    print(name, cos.min())
    assert cos.min() >= 0.999, cos


@pytest.mark.parametrize("name,layers,mode", [("qwen3-0.6b", 28, "bf16"), ("xlmr-large", 24, "16f")])
def test_full_depth(name, layers, mode, model_root):
    """All layers of a model against the exact plan.  Four products a layer, each off
    by up to 0.03 of itself, add up to at most 0.03 sqrt(4 x 28) = 0.32 of a row:
    cosine 1 - 0.32^2 / 2 = 0.95."""
    d = synth.ensure_model(synth.spec(name, n_layers=layers, vocab=8192), model_root)
    seqs = synth.token_batch(name, seed=1, batch=6, vocab=8192)
    out = {}
    for i8, kw in ((False, dict(gemm_mode="f32", weight_dtype="f32")),
                   (True, dict(gemm_mode=mode, weight_dtype="file"))):
        m = native.B200Model(d, linear_i8=i8, **kw)
        try:
            out[i8] = m.encode_batch(seqs)
        finally:
            m.close()
    cos = cos_rows(out[False], out[True])
    print(name, cos.min())
    assert cos.min() >= 0.95, cos
