"""Source rules of the 8-bit integer kernels (CPU only, reads the sources)."""

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ffwd_b200",
                    "csrc")


def test_no_read_only_loads():
    """A read-only (non-coherent) load promises that nothing writes the data while
    the kernel runs.  These kernels run, as dependent launches, while the
    stream's previous kernel may still be writing their rows, codes, scales and
    weights, and the LayerNorm writes its rows in place."""
    files = sorted(glob.glob(os.path.join(CSRC, "int8*")))
    assert len(files) >= 6
    for path in files:
        text = open(path).read()
        assert not re.search(r"__ldg|__ldcs|ld\.global[.\w]*\.nc|__restrict__", text), path


def test_every_device_error_has_a_text():
    """The host names each code that a kernel can record."""
    enum = re.search(r"enum DevError : int \{(.*?)\};", open(os.path.join(CSRC, "ptx.cuh")).read(),
                     re.S).group(1)
    codes = [c for c in re.findall(r"\b(kErr\w+) =", enum) if c != "kErrNone"]
    assert "kErrBadPosition" in codes
    engine = open(os.path.join(CSRC, "engine.cu")).read()
    text = engine[engine.index("int check_err(Device &D) {"):]
    text = text[:text.index("\n}\n")]
    assert [c for c in codes if c not in text] == []
