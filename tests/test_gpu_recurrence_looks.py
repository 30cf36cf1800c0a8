"""Tiles of the gated recurrence that give up waiting, forced by a limit of a few looks: every value is the one
of an unhurried call or NaN, those behind the tile that gave up among them."""
import pytest
import torch

from reimagined_amd import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.fixture
def limit():
    looks = _lib.lib().nsosx_gated_recurrence_looks
    before = looks(-1)
    yield looks
    looks(before)


def right_or_nan(got, want):
    """How many are NaN; every other one has want's bits."""
    lost = got.isnan()
    assert torch.equal(torch.where(lost, want, got), want)
    return int(lost.sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bounds", [[0, 40000], [0, 1000, 1000, 1003, 9000, 20500, 40000]], ids=["one", "some"])
def test_gives_up(dev, limit, dtype, bounds):
    torch.manual_seed(3)
    t, d, s = bounds[-1], 520, len(bounds) - 1
    x, rg, ig, dy = (torch.randn((t, d), device=dev).to(dtype) for _ in range(4))
    lam = torch.randn(d, device=dev) - 6.0  # (states that last for thousands of tokens)
    cu = torch.tensor(bounds, dtype=torch.int32, device=dev)
    h0, dfinal = (torch.randn((s, d), device=dev) for _ in range(2))
    forward = lambda: ops.gated_recurrence(x, rg, ig, lam, cu, initial_state=h0, want_carry=True)
    y, final, carry = forward()
    back = lambda: ops.gated_recurrence_backward(dy, x, rg, ig, lam, cu, carry, initial_state=h0, dfinal=dfinal)
    want = back()
    assert torch.isfinite(y).all() and all(torch.isfinite(g).all() for g in want.values())
    lost = [0, 0]
    for looks in (0, 0, 0, 1, 2, 5, 30):
        limit(looks)
        py, pfinal, pcarry = forward()
        got = back()
        torch.cuda.synchronize()
        lost[0] += right_or_nan(py, y) + right_or_nan(pfinal, final)
        lost[1] += sum(right_or_nan(got[k], want[k]) for k in want)
        # (what the forward kept, for the gradients: NaN or right as well, but for rows no sequence enters)
        right_or_nan(pcarry, carry)
    assert lost[0] > 0 and lost[1] > 0  # some did give up
    limit(1 << 22)
    assert torch.equal(forward()[0], y) and all(torch.equal(g, want[k]) for k, g in back().items())
