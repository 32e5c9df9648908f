"""Empty calls of the 8-bit integer entries (M = 0): an empty tensor has no
address, and the call is one all the same.  What does not hang on the rows is
still checked."""

import pytest

from ffwd_b200 import native
from test_int8_host import gated, gemm, heads, mat, qkv, quantise


@pytest.mark.parametrize("null", [None, 0])
def test_tensors_without_an_address(null):
    quantise(M=0, x_ptr=null, q_ptr=null, scale_ptr=null)
    quantise(M=0, x_ptr=null, q_ptr=null, scale_ptr=null, norm_ptr=1 << 20, eps=1e-6)
    gemm(M=0, x_ptr=null, xs_ptr=null, y_ptr=null)
    gated(M=0, x_ptr=null, xs_ptr=null, h_ptr=null)
    qkv(M=0, x_ptr=null, xs_ptr=null, out_ptr=null)
    qkv(h=heads(pos_ptr=null), M=0, x_ptr=null, xs_ptr=null, out_ptr=null)


@pytest.mark.parametrize("call,kw,text", [
    (quantise, dict(K=0), "invalid arguments"),
    (quantise, dict(dtype="int8"), "is not one of"),
    (quantise, dict(ldq=104), "multiple of 16"),
    (gemm, dict(w=mat(q_ptr=None)), "invalid weights"),
    (gemm, dict(ldx=96), "at least 100"),
    (gemm, dict(ldy=63), "at least 64"),
    (gemm, dict(act="relu"), "is not one of"),
    (gated, dict(up=mat(cols=99)), "gate is 64 x 100, up 64 x 99"),
    (qkv, dict(h=heads(cos_ptr=None)), "invalid heads"),
    (qkv, dict(h=heads(head_dim=96)), "head_dim 96"),
])
def test_still_refused(call, kw, text):
    with pytest.raises(native.FfwdError, match=text):
        call(M=0, **kw)
