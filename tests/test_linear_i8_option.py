"""Which plan a load gets: the caller's own choice, else the process's switch.

An exact plan with 8-bit projections is refused before anything touches a GPU,
so the refusal shows on any machine what a load was asked for."""

import threading

import pytest

from ffwd_b200 import native, synth
from helpers import small_spec

REFUSED = "16-bit plan"


@pytest.fixture(scope="module")
def dirs(model_root):
    """(pooled, late) models whose f32 mode is an exact plan."""
    return (synth.ensure_model(small_spec("bert-tanh-1l"), model_root),
            synth.ensure_model(small_spec("qwen3-late-f32-1l"), model_root))


@pytest.fixture(autouse=True)
def _defaults():
    L = native.lib()
    L.ffwd_b200_set_weights_default()
    L.ffwd_b200_set_fast_gemm(b"f32")
    L.ffwd_b200_set_linear_i8(0)
    yield
    L.ffwd_b200_set_linear_i8(0)


def eight_bit(cls, d, **kw):
    """Whether a load under f32 asks for 8-bit projections (it is refused then)."""
    try:
        cls(d, **kw).close()
    except native.FfwdError as e:
        return REFUSED in str(e)
    return False


@pytest.mark.parametrize("late", [False, True])
def test_the_switch_holds_for_all_next_loads(dirs, late):
    cls = native.B200Late if late else native.B200Model
    L = native.lib()
    assert not eight_bit(cls, dirs[late])
    L.ffwd_b200_set_linear_i8(1)
    assert eight_bit(cls, dirs[late])
    assert eight_bit(cls, dirs[late])  # a load leaves the switch as it is
    L.ffwd_b200_set_linear_i8(0)
    assert not eight_bit(cls, dirs[late])


@pytest.mark.parametrize("late", [False, True])
@pytest.mark.parametrize("switch", [0, 1])
def test_a_load_with_its_own_choice(dirs, late, switch):
    """It has that plan whatever the switch says, and leaves the switch alone."""
    cls = native.B200Late if late else native.B200Model
    native.lib().ffwd_b200_set_linear_i8(switch)
    for own in (True, False, True):
        assert eight_bit(cls, dirs[late], linear_i8=own) == own
        assert eight_bit(cls, dirs[late]) == bool(switch)


def test_loads_of_two_threads(dirs):
    """A thread that asks for 8 bits and one that asks for nothing get just that."""
    n, got = 300, {}

    def work(key, **kw):
        got[key] = [eight_bit(native.B200Model, dirs[0], **kw) for _ in range(n)]

    ts = [threading.Thread(target=work, args=("on",), kwargs=dict(linear_i8=True)),
          threading.Thread(target=work, args=("default",))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert got["on"] == [True] * n and got["default"] == [False] * n


def test_choices_out_of_range():
    L = native.lib()
    for f in (L.ffwd_b200_load_linear, L.ffwd_b200_late_load_linear):
        assert not f(b"/nonexistent", 2)
        assert "linear_i8" in native.last_error()
