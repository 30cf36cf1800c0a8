"""The gated recurrence where decays multiply to less than float32 holds: large finite states are forgotten
wherever they lie among the tiles' cuts, and fade by the bits that they have."""
import numpy as np
import pytest
import torch

import train_ref as ref
from reimagined_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
# A product of decays below 2^-126 is off by half of 2^-149 at each of at most 92 roundings (16 tokens of a wave, 8
# waves, 4 tiles, 64 groups of them), or held at 2^-149, and a state that it multiplies by as much of that state.
FAR = 2.0**-143


def near(got, want, lim, dtype, what):
    got = got.double().cpu().numpy()
    bound = lim + ref.HALF_STEP[dtype] * np.abs(want) * (1 + 2.0**-7) + 1e-37
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / bound)))


def make(dev, dtype, bounds, lam):
    rng = np.random.default_rng([len(bounds), bounds[-1]])
    t, d = bounds[-1], lam.size
    c = {k: torch.from_numpy(rng.standard_normal((t, d)).astype(np.float32)).to(DT[dtype]).to(dev)
         for k in ("x", "rg", "ig", "dy")}
    c["lam"] = torch.from_numpy(lam.astype(np.float32)).to(dev)
    c["cu"] = torch.tensor(bounds, dtype=torch.int32, device=dev)
    for k in ("h0", "dfinal"):
        c[k] = torch.from_numpy(rng.standard_normal((len(bounds) - 1, d)).astype(np.float32)).to(dev)
    return c


def definition(c):
    n = {k: v.double().cpu().numpy() for k, v in c.items()}
    return ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"].astype(int), 8.0, n["h0"]), n


# open gates of 2^-1 to 2^-92 a token: products of 8 and 16 tokens on either side of 2^-126 and 2^-149
LAM = np.linspace(-2.5, 7.9, 40)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bounds", [[0, 700], [0, 131, 140, 140, 2100]], ids=["one", "some"])
def test_large_states_fade(dev, dtype, bounds):
    c = make(dev, dtype, bounds, LAM)
    big = 1.0e38
    c["h0"] = c["h0"].sign() * big
    for t in (17, 100, 250, 333, 600):  # and inputs as large, at several places of a wave and a tile
        c["x"][t] = big if t % 2 else -big
    y, final = ops.gated_recurrence(c["x"], c["rg"], c["ig"], c["lam"], c["cu"], initial_state=c["h0"])
    want, _ = definition(c)
    near(y, want.h, want.eh + FAR * big, dtype, "y")
    near(final, want.final, want.efinal + FAR * big, "f32", "final")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bounds", [[0, 700], [0, 131, 140, 140, 2100]], ids=["one", "some"])
def test_large_gradients_fade(dev, dtype, bounds):
    c = make(dev, dtype, bounds, LAM)
    big = 1.0e36
    c["dfinal"] = c["dfinal"].sign() * big
    for t in (17, 100, 250, 333, 600):
        c["dy"][t] = big if t % 2 else -big
    _, _, carry = ops.gated_recurrence(c["x"], c["rg"], c["ig"], c["lam"], c["cu"], initial_state=c["h0"],
                                       want_carry=True)
    got = ops.gated_recurrence_backward(c["dy"], c["x"], c["rg"], c["ig"], c["lam"], c["cu"], carry,
                                        initial_state=c["h0"], dfinal=c["dfinal"])
    want, n = definition(c)
    grads = want.backward(n["dy"], n["dfinal"])
    # what is off of dh meets factors below 1, x (8 at most), and a g h (g up to 64, h up to 8)
    for k in ("dx", "drg", "dig"):
        near(got[k], grads[k][0], grads[k][1] + 512 * FAR * big, dtype, k)
    near(got["dinitial"], grads["dinitial"][0], grads["dinitial"][1] + FAR * big, "f32", "dinitial")
    near(got["dlam"], *grads["dlam"], "f32", "dlam")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1, 7, 8, 15, 64, 127])
def test_cuts_do_not_show(dev, dtype, shift):
    """A sequence behind rows of no sequence, so that the tiles cut it elsewhere: what follows a large state has
    the same values, but for roundings."""
    bounds = [0, 400]
    c = make(dev, dtype, bounds, LAM)
    c["h0"] = c["h0"].sign() * 1.0e38
    p = dict(c)
    for k in ("x", "rg", "ig"):
        p[k] = torch.cat([torch.zeros((shift, LAM.size), dtype=DT[dtype], device=dev), c[k]])
    p["cu"] = c["cu"] + shift
    want, _ = definition(c)
    y, _ = ops.gated_recurrence(p["x"], p["rg"], p["ig"], p["lam"], p["cu"], initial_state=p["h0"])
    near(y[shift:], want.h, want.eh + FAR * 1.0e38, dtype, "y")
