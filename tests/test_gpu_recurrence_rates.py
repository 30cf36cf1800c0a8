"""The gated recurrence at other rates than 8 and decays from nearly 1 to nearly 0, where the kernels take the
longer of their two forms of 1 - a^2: operators, step and layer against float64."""
import numpy as np
import pytest
import torch

import test_gpu_recurrent_layer as whole
import train_ref as ref
from reimagined_amd import ops
from reimagined_amd.layers import RecurrentLayer
from test_gpu_recurrence import make, near

pytestmark = pytest.mark.gpu

RATES = [0.01, 1.0, 2.5, 40.0]


def spread(c, n, kind, dev):
    """Decays of all channels as make() has them, wide apart, or one strong one in each run of channels."""
    d = n["lam"].size
    rng = np.random.default_rng(d)
    lam = n["lam"].astype(np.float32)
    if kind == "wide":
        lam = rng.uniform(-7.0, 5.0, d).astype(np.float32)
    elif kind == "one":
        lam[5::64] = 1.0
    c["lam"], n["lam"] = torch.from_numpy(lam).to(dev), lam.astype(np.float64)


@pytest.mark.parametrize("rate", RATES)
@pytest.mark.parametrize("kind", ["weak", "wide", "one"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,d,initial", [([129], 70, False), ([40, 0, 300, 1, 1, 77], 131, True), ([3] * 90, 64, True)],
                         ids=["one", "ragged", "short"])
def test_operators(dev, rate, kind, dtype, lens, d, initial):
    c, n = make(dev, lens, d, dtype, initial)
    spread(c, n, kind, dev)
    want = ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"], rate, n["h0"])
    a = (c["x"], c["rg"], c["ig"], c["lam"])
    y, final, carry = ops.gated_recurrence(*a, c["cu"], rate=rate, initial_state=c["h0"], want_carry=True)
    near(y, want.h, want.eh, dtype, "y")
    near(final, want.final, want.efinal, what="final")
    got = ops.gated_recurrence_backward(c["dy"], *a, c["cu"], carry, rate=rate, initial_state=c["h0"],
                                        dfinal=c["dfinal"])
    grads = want.backward(n["dy"], n["dfinal"])
    for name, g in got.items():
        near(g, *grads[name], dtype=dtype if name in ("dx", "drg", "dig") else "f32", what=name)


@pytest.mark.parametrize("rate", RATES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_step(dev, rate, dtype):
    rows = 37
    c, n = make(dev, [1] * rows, 200, dtype, True)
    spread(c, n, "wide", dev)
    want = ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"], rate, n["h0"])
    state = c["h0"].clone()
    y = ops.gated_recurrence_step(c["x"], c["rg"], c["ig"], c["lam"], state, rate=rate)
    near(y, want.h, want.eh, dtype, "y")
    near(state, want.final, want.efinal, what="state")


@pytest.mark.parametrize("rate", [1.0, 20.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer(dev, rate, dtype):
    rng = np.random.default_rng(7)
    n = lambda *s: rng.standard_normal(s).astype(np.float32)
    layer = RecurrentLayer(dict(w_in=0.1 * n(240, 64), w_out=0.1 * n(64, 80), lam=2.0 * n(80) - 2.0, rate=rate), dev)
    lens = [150, 0, 61]
    cu, rnd = whole.batch(dev, lens, 64, dtype, 3, 5)
    x, delta, dout, dres = rnd(), rnd(), rnd(0.1), rnd(0.1)
    fwd = layer.forward(x, cu, delta, train=True)
    rec = whole.check_forward(layer, x, delta, cu, None, fwd, dtype)
    g = layer.backward(fwd, dout, dres)
    whole.check_backward(layer, fwd, rec, dout, dres, None, g, dtype)
    # and the decode step at that rate: the packed pass's first tokens
    state = layer.new_decode_state(1, dev)
    for t in range(3):
        layer.step(x[t:t + 1], state, delta[t:t + 1])
        whole.near(state, rec.h[t:t + 1], rec.eh[t:t + 1], what="state")
