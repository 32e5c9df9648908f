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
