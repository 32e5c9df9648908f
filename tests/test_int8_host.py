"""Refusals of the 8-bit integer entries that are decided on the host, before
anything touches a GPU (addresses below are never followed)."""

import ctypes

import pytest

from ffwd_b200 import native

A = 1 << 20  # an aligned address


def mat(**kw):
    a = dict(q_ptr=A, scale_ptr=A, rows=64, cols=100, ld=112)
    a.update(kw)
    return native.i8_mat(**a)


def heads(**kw):
    a = dict(n_heads=2, n_kv_heads=1, head_dim=64, pos_ptr=A, cos_ptr=A, sin_ptr=A, n_pos=8,
             q_norm_ptr=A, k_norm_ptr=A, eps=1e-6)
    a.update(kw)
    return native.i8_heads(**a)


def quantise(**kw):
    a = dict(x_ptr=A, dtype="bf16", ldx=100, q_ptr=A, ldq=112, scale_ptr=A, M=3, K=100)
    a.update(kw)
    native.quantize_i8(**a)


def gemm(w=None, **kw):
    a = dict(x_ptr=A, ldx=112, xs_ptr=A, M=3, y_ptr=A, dtype="bf16", ldy=64)
    a.update(kw)
    native.gemm_i8(w if w is not None else mat(), **a)


def gated(gate=None, up=None, **kw):
    a = dict(x_ptr=A, ldx=112, xs_ptr=A, M=3, h_ptr=A, dtype="f16", ldh=64)
    a.update(kw)
    native.gated_i8(gate or mat(), up or mat(), **a)


def qkv(w=None, h=None, **kw):
    a = dict(x_ptr=A, ldx=112, xs_ptr=A, M=3, out_ptr=A, dtype="f32", ldo=256)
    a.update(kw)
    native.qkv_i8(w or mat(rows=256), h or heads(), **a)


@pytest.mark.parametrize("call,kw,text", [
    (quantise, dict(x_ptr=None), "invalid arguments"),
    (quantise, dict(q_ptr=None), "invalid arguments"),
    (quantise, dict(scale_ptr=None), "invalid arguments"),
    (quantise, dict(M=-1), "invalid arguments"),
    (quantise, dict(K=0), "invalid arguments"),
    (quantise, dict(dtype="int8"), "is not one of"),
    (quantise, dict(x_ptr=A + 1), "element alignment"),
    (quantise, dict(ldx=99), "stride of at least 100"),
    (quantise, dict(ldq=104), "multiple of 16"),
    (quantise, dict(ldq=96), "at least 100"),
    (quantise, dict(q_ptr=A + 8), "16-byte aligned"),
    (quantise, dict(scale_ptr=A + 2), "4-byte"),
    (quantise, dict(norm_ptr=A, eps=0.0), "positive eps"),
    (quantise, dict(norm_ptr=A, eps=float("nan")), "positive eps"),
    (gemm, dict(w=mat(q_ptr=None)), "invalid weights"),
    (gemm, dict(w=mat(scale_ptr=None)), "invalid weights"),
    (gemm, dict(w=mat(rows=0)), "invalid weights"),
    (gemm, dict(w=mat(cols=0)), "invalid weights"),
    (gemm, dict(w=mat(cols=131072, ld=131072)), "at most 131071"),
    (gemm, dict(w=mat(ld=104)), "multiple of 16"),
    (gemm, dict(w=mat(q_ptr=A + 4)), "16-byte aligned"),
    (gemm, dict(w=mat(bias_ptr=A + 1)), "4-byte"),
    (gemm, dict(x_ptr=None), "invalid arguments"),
    (gemm, dict(xs_ptr=None), "invalid arguments"),
    (gemm, dict(M=-2), "invalid arguments"),
    (gemm, dict(M=(1 << 30) + 1), "invalid arguments"),
    (quantise, dict(M=(1 << 30) + 1), "invalid arguments"),
    (gemm, dict(ldx=96), "at least 100"),
    (gemm, dict(x_ptr=A + 1), "16-byte aligned"),
    (gemm, dict(y_ptr=None), "invalid arguments"),
    (gemm, dict(y_ptr=A + 1), "element alignment"),
    (gemm, dict(ldy=63), "at least 64"),
    (gemm, dict(err_ptr=A + 2), "error word"),
    (gemm, dict(act="relu"), "is not one of"),
    (gemm, dict(accumulate=True), "only f32"),
    (gated, dict(up=mat(rows=65)), "gate is 64 x 100, up 65 x 100"),
    (gated, dict(up=mat(cols=99)), "gate is 64 x 100, up 64 x 99"),
    (gated, dict(up=mat(ld=100)), "multiple of 16"),
    (gated, dict(act="none"), "gate activation"),
    (gated, dict(h_ptr=None), "invalid arguments"),
    (qkv, dict(h=heads(n_heads=0)), "invalid heads"),
    (qkv, dict(h=heads(pos_ptr=None)), "invalid heads"),
    (qkv, dict(h=heads(cos_ptr=None)), "invalid heads"),
    (qkv, dict(h=heads(n_pos=0)), "invalid heads"),
    (qkv, dict(h=heads(head_dim=96)), "head_dim 96"),
    (qkv, dict(h=heads(n_heads=3)), "do not make 256 rows"),
    (qkv, dict(h=heads(eps=0.0)), "positive eps"),
    (qkv, dict(h=heads(sin_ptr=A + 4)), "16-byte alignment"),
    (qkv, dict(ldo=255), "at least 256"),
])
def test_refused_on_the_host(call, kw, text):
    with pytest.raises(native.FfwdError, match=text):
        call(**kw)


def test_null_descriptors():
    L = native.lib()
    assert L.ffwd_b200_gemm_i8(None, A, 112, A, 1, A, 0, 64, 0, 0, None, None) == -1
    assert L.ffwd_b200_qkv_i8(ctypes.byref(mat(rows=256)), None, A, 112, A, 1, A, 0, 256, None,
                              None) == -1
    assert L.ffwd_b200_gemm_i8(ctypes.byref(mat()), A, 112, A, 1, A, 3, 64, 0, 0, None, None) == -1
    assert L.ffwd_b200_gemm_i8(ctypes.byref(mat()), A, 112, A, 1, A, 0, 64, 9, 0, None, None) == -1


def test_no_rows_is_an_empty_call():
    quantise(M=0)
    gemm(M=0)
    gated(M=0)
    qkv(M=0)
