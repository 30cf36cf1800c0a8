"""Views of the gated recurrence over states and rates are refused (CPU only): the C entries on placeholder
addresses that no check dereferences."""
import pytest

from reimagined_amd import _lib

P = 1 << 30  # never dereferenced, far apart
LAM, CU, H0, CARRY, DFINAL, WS = (P * i for i in range(20, 26))


def refused(fn, *args):
    lib = _lib.lib()
    assert getattr(lib, fn)(*args) == 1
    return lib.nsosx_last_error().decode()


def forward(y, ys=8, h0=H0):
    return (P, 8, 2 * P, 8, 3 * P, 8, LAM, 8.0, CU, 2, 4, 8, 0, h0, 1, y, ys, None, None, WS, None)


# (states [2, 8] and rates [8] f32: 64 and 32 bytes; four rows of 32 bytes, 4 ys apart: of the last of H0's the
# first three end before the states, the fourth lies in them)
@pytest.mark.parametrize("y,ys", [(H0, 8), (H0 + 60, 8), (H0 - 3 * 32 - 28, 8), (H0 - 384, 96), (H0 - 448, 40),
                                  (LAM, 8), (LAM + 28, 8), (LAM - 124, 8)])
def test_forward(y, ys):
    assert "y overlaps an input" in refused("nsosx_gated_recurrence", *forward(y, ys))


def backward(dx=P * 10, drg=P * 11, dig=P * 12, s=8):
    return (P, 8, 2 * P, 8, 3 * P, 8, 4 * P, 8, LAM, 8.0, CU, 2, 4, 8, 0, H0, CARRY, DFINAL, 1, dx, s, drg, s, dig, s,
            13 * P, 14 * P, WS, None)


@pytest.mark.parametrize("where", [H0, H0 + 60, DFINAL + 4, CARRY + 28, CARRY - 124, LAM, LAM - 100])
@pytest.mark.parametrize("which", ["dx", "drg", "dig"])
def test_backward(which, where):
    assert "a gradient overlaps an input" in refused("nsosx_gated_recurrence_backward", *backward(**{which: where}))


def step(x=P, xs=8, rg=2 * P, ig=3 * P, dt=0, state=H0, out=DFINAL, y=P * 10, ys=8):
    return (x, xs, rg, 8, ig, 8, LAM, 8.0, 4, 8, dt, state, out, y, ys, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=DFINAL + 4), "state_out overlaps"), (dict(rg=DFINAL - 96), "state_out overlaps"),
    (dict(ig=DFINAL, dt=1), "state_out overlaps"), (dict(x=DFINAL, xs=16), "state_out overlaps"),
    (dict(y=DFINAL + 32), "state_out overlaps"), (dict(y=DFINAL, dt=1), "state_out overlaps"),
    (dict(y=H0, ys=16), "y overlaps state"), (dict(y=H0 + 124), "y overlaps state"),
])
def test_step(kw, text):
    assert text in refused("nsosx_gated_recurrence_step", *step(**kw))
