"""The gated recurrence, its gradients and its step against float64: ragged batches across the tiles'
borders, empty sequences, rows of no sequence, odd widths, column slices, captured calls."""
import numpy as np
import pytest
import torch

import train_ref as ref
from reimagined_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def tensor(a, dtype, dev):
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(DT[dtype])
    return t.to(dev), t.double().numpy()


def make(dev, lens, d, dtype, initial, seed=0, rest=0):
    rng = np.random.default_rng([len(lens), sum(lens), d, seed])
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    t = int(cu[-1]) + rest
    c = {"cu": torch.from_numpy(cu).to(dev)}
    n = {"cu": cu}
    for name, scale in (("x", 1.0), ("rg", 1.5), ("ig", 1.5), ("dy", 0.1)):
        c[name], n[name] = tensor(scale * rng.standard_normal((t, d)), dtype, dev)
    lam = np.log(np.expm1(-np.log(rng.uniform(0.9, 0.999, d)) / 8.0))
    c["lam"], n["lam"] = tensor(lam, "f32", dev)
    s = len(lens)
    for name, scale in (("h0", 1.0), ("dfinal", 0.1)):
        c[name], n[name] = tensor(scale * rng.standard_normal((s, d)), "f32", dev) if initial else (None, None)
    return c, n


def near(got, want, lim, dtype="f32", what=""):
    got = got.double().cpu().numpy()
    bound = lim + ref.HALF_STEP[dtype] * np.abs(want) * (1 + 2.0**-7) + 1e-37
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / bound)))


def forward(c, **kw):
    return ops.gated_recurrence(c["x"], c["rg"], c["ig"], c["lam"], c["cu"], initial_state=c["h0"],
                                want_carry=True, **kw)


def backward(c, carry, **kw):
    return ops.gated_recurrence_backward(c["dy"], c["x"], c["rg"], c["ig"], c["lam"], c["cu"], carry,
                                         initial_state=c["h0"], dfinal=c["dfinal"], **kw)


# one token; a tile's border inside, at and behind a sequence; many sequences in a tile; empty ones first,
# last and in a row; a sequence over many tiles; more sequences than threads
LENS = [[1], [2], [127], [128], [129], [1000], [5, 0, 0, 300, 0, 1, 1, 128, 0], [0, 0, 3], [64] * 9,
        [1] * 300, [0] * 700 + [130, 5], [257, 255], [3] * 1100]


@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}x{sum(v)}")
@pytest.mark.parametrize("d", [1, 2, 67, 129, 256])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("initial", [False, True])
def test_against_float64(dev, lens, d, dtype, initial):
    if sum(lens) * d > 300000 or (len(lens) > 600 and d > 67):
        d = 30 + d % 2
    c, n = make(dev, lens, d, dtype, initial)
    want = ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"], 8.0, n["h0"])
    y, final, carry = forward(c)
    near(y, want.h, want.eh, dtype, "y")
    near(final, want.final, want.efinal, what="final")
    got = backward(c, carry)
    grads = want.backward(n["dy"], n["dfinal"])
    assert ("dinitial" in got) == initial
    for name, g in got.items():
        near(g, *grads[name], dtype=dtype if name in ("dx", "drg", "dig") else "f32", what=name)
    # the same bits every time
    y2, final2, carry2 = forward(c)
    again = backward(c, carry2)
    assert torch.equal(y, y2) and torch.equal(final, final2)
    assert all(torch.equal(got[k], again[k]) for k in got)
    # and of y and the final states without the kept ones
    y3, none = ops.gated_recurrence(c["x"], c["rg"], c["ig"], c["lam"], c["cu"], initial_state=c["h0"],
                                    want_final=False)
    assert none is None and torch.equal(y, y3)


@pytest.mark.parametrize("d", [2050, 4200, 8200])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_wide(dev, d, dtype):
    """Many blocks of channels (the last one narrow), several tiles of each, against the same channels in
    a narrow call of their own."""
    c, _ = make(dev, [300, 500], d, dtype, True)
    y, final, carry = forward(c)
    got = backward(c, carry)
    for lo, hi in ((0, 64), (2000, 2050), (d - 70, d), (d - 1, d)):
        p = {k: v if k == "cu" else v[..., lo:hi].contiguous() for k, v in c.items()}
        py, pfinal, pcarry = forward(p)
        want = backward(p, pcarry)
        assert torch.equal(y[:, lo:hi], py) and torch.equal(final[:, lo:hi], pfinal)
        for k in want:
            assert torch.equal(got[k][..., lo:hi], want[k]), k


@pytest.mark.parametrize("seqs", [2046, 2047, 2048, 5000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_sequences(dev, seqs, dtype):
    """More bounds than the kernels keep on the chip."""
    c, n = make(dev, [(7 * i) % 4 for i in range(seqs)], 20, dtype, True)
    want = ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"], 8.0, n["h0"])
    y, final, carry = forward(c)
    near(y, want.h, want.eh, dtype, "y")
    near(final, want.final, want.efinal, what="final")
    grads = want.backward(n["dy"], n["dfinal"])
    for name, g in backward(c, carry).items():
        near(g, *grads[name], dtype=dtype if name in ("dx", "drg", "dig") else "f32", what=name)


def test_long_sequence(dev):
    """Many tiles behind one another (a state that crosses hundreds of them)."""
    c, n = make(dev, [40000, 7], 6, "f32", True)
    want = ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"], 8.0, n["h0"])
    y, final, carry = forward(c)
    near(y, want.h, want.eh, what="y")
    got = backward(c, carry)
    for name, (g, lim) in want.backward(n["dy"], n["dfinal"]).items():
        near(got[name], g, lim, what=name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("before,behind", [(0, 1), (0, 300), (5, 0), (200, 77)])
def test_rows_of_no_sequence(dev, dtype, before, behind):
    """Rows before the first and behind the last sequence: zeros in fresh tensors, left as they were in
    given ones, and whatever they hold (NaN here) reaches nothing."""
    lens, d = [100, 0, 131], 70
    c, n = make(dev, lens, d, dtype, True)
    t = sum(lens)
    p = dict(c)
    for name in ("x", "rg", "ig", "dy"):
        p[name] = torch.full((before + t + behind, d), float("nan"), dtype=DT[dtype], device=dev)
        p[name][before:before + t] = c[name]
    p["cu"] = c["cu"] + before
    py, pfinal, pcarry = forward(p)
    got = backward(p, pcarry)
    inner = slice(before, before + t)
    want = ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"], 8.0, n["h0"])
    grads = want.backward(n["dy"], n["dfinal"])
    for k, a, w, lim in [("y", py, want.h, want.eh)] + [(k, got[k], *grads[k]) for k in ("dx", "drg", "dig")]:
        assert not a[:before].any() and not a[before + t:].any(), k
        near(a[inner], w, lim, dtype, k)
    near(pfinal, want.final, want.efinal, what="final")
    for k in ("dlam", "dinitial"):
        near(got[k], *grads[k], what=k)
    wide = torch.full((before + t + behind, 4 * d), 7.0, dtype=DT[dtype], device=dev)
    views = [wide[:, i * d:(i + 1) * d] for i in range(4)]
    ops.gated_recurrence(p["x"], p["rg"], p["ig"], p["lam"], p["cu"], initial_state=p["h0"], out=views[0])
    backward(p, pcarry, out=views[1:])
    for v, a in zip(views, (py, got["dx"], got["drg"], got["dig"])):
        assert torch.equal(v[inner], a[inner])
    assert (wide[:before] == 7.0).all() and (wide[before + t:] == 7.0).all()


@pytest.mark.parametrize("d", [5, 64, 131])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_column_slices(dev, d, dtype):
    """Inputs as columns of one projection, at odd offsets."""
    c, _ = make(dev, [50, 200], d, dtype, False)
    y, final, carry = forward(c)
    want = backward(c, carry)
    wide = torch.full((250, 3 * d + 3), float("nan"), dtype=DT[dtype], device=dev)
    p = dict(c)
    for i, name in enumerate(("x", "rg", "ig")):
        p[name] = wide[:, i * (d + 1):i * (d + 1) + d]
        p[name].copy_(c[name])
    py, pfinal, pcarry = forward(p)
    assert torch.equal(py, y) and torch.equal(pfinal, final)
    got = backward(p, pcarry)
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_not_finite_stays_in_its_sequence(dev):
    """A NaN or an infinity in one sequence reaches no other one, forward or backward."""
    lens, d = [40, 60, 200, 30], 33
    c, _ = make(dev, lens, d, "f32", True)
    y, final, carry = forward(c)
    want = backward(c, carry)
    p = {k: v.clone() for k, v in c.items()}
    p["x"][45, 3] = float("inf")
    p["rg"][50, 4] = float("nan")
    p["dy"][90, 5] = float("nan")
    p["h0"][1, 6] = float("inf")
    p["dfinal"][1, 7] = float("nan")
    py, pfinal, pcarry = forward(p)
    got = backward(p, pcarry)
    bad = slice(40, 100)
    for a, b in ((py, y), (got["dx"], want["dx"]), (got["drg"], want["drg"]), (got["dig"], want["dig"])):
        assert torch.equal(a[:40], b[:40]) and torch.equal(a[100:], b[100:])
        assert not torch.isfinite(a[bad]).all()
    keep = [0, 2, 3]
    assert torch.equal(pfinal[keep], final[keep]) and torch.equal(got["dinitial"][keep], want["dinitial"][keep])
    assert torch.isnan(py[50:100, 4]).all() and torch.isinf(py[45:100, 3]).all()


def test_extreme_gates(dev):
    """Closed, open and saturated gates, decays of nearly 0 and nearly 1: finite values and gradients."""
    v = torch.tensor([0.0, 1e-3, -1e-3, 20.0, -20.0, 89.0, -89.0, 1e4, -1e4, float("inf"), float("-inf")])
    rg, ig = torch.meshgrid(v, v, indexing="ij")
    rg, ig = rg.reshape(-1, 1).repeat(1, 6).to(dev), ig.reshape(-1, 1).repeat(1, 6).to(dev)
    t = rg.shape[0]
    lam = torch.tensor([-100.0, -30.0, -4.0, 0.0, 4.0, 30.0], device=dev)
    x = torch.randn((t, 6), device=dev).clamp(-8, 8)
    cu = torch.tensor([0, t], dtype=torch.int32, device=dev)
    y, final, carry = ops.gated_recurrence(x, rg, ig, lam, cu, want_carry=True)
    g = ops.gated_recurrence_backward(torch.ones_like(x), x, rg, ig, lam, cu, carry)
    assert torch.isfinite(y).all() and torch.isfinite(final).all()
    for k, a in g.items():
        assert torch.isfinite(a).all(), k
    big = torch.nan_to_num(rg.double().cpu(), posinf=1e4, neginf=-1e4).numpy()
    big2 = torch.nan_to_num(ig.double().cpu(), posinf=1e4, neginf=-1e4).numpy()
    want = ref.Recurrence(x.double().cpu().numpy(), big, big2, lam.double().cpu().numpy(), [0, t], 8.0, None)
    # The exponential, root and product units read a g below 2^-126, float32's normal numbers, as zero:
    # beta = sqrt(2 g) is then off by up to sqrt(2^-125), and so are g / beta = sqrt(g / 2) and what they
    # multiply: x <= 8 here, and sums of at most t tokens (lam = -100: g = 3e-43, y = 1e-22).
    below = t * 8 * 2.0**-62.5
    near(y, want.h, want.eh + below, what="y")
    grads = want.backward(np.ones((t, 6)))
    for k in ("dx", "dig", "drg"):
        near(g[k], grads[k][0], grads[k][1] + below, what=k)


def test_no_tokens(dev):
    d = 9
    x = torch.empty((0, d), device=dev)
    cu = torch.zeros(4, dtype=torch.int32, device=dev)
    lam, h0, dfin = torch.zeros(d, device=dev), torch.randn((3, d), device=dev), torch.randn((3, d), device=dev)
    y, final, carry = ops.gated_recurrence(x, x, x, lam, cu, initial_state=h0, want_carry=True)
    assert y.shape == (0, d) and torch.equal(final, h0)
    g = ops.gated_recurrence_backward(x, x, x, x, lam, cu, carry, initial_state=h0, dfinal=dfin)
    assert torch.equal(g["dinitial"], dfin) and not g["dlam"].any()


@pytest.mark.parametrize("rows,d", [(1, 1), (1, 2048), (3, 67), (8, 512), (33, 1001), (130, 256), (1000, 130)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_step(dev, rows, d, dtype):
    c, n = make(dev, [1] * rows, d, dtype, True)
    want = ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"], 8.0, n["h0"])
    state, out = c["h0"].clone(), torch.empty_like(c["h0"])
    y = ops.gated_recurrence_step(c["x"], c["rg"], c["ig"], c["lam"], state, state_out=out)
    assert torch.equal(state, c["h0"])
    near(out, want.final, want.efinal, what="state")
    near(y, want.h, want.eh, dtype, "y")
    y2 = ops.gated_recurrence_step(c["x"], c["rg"], c["ig"], c["lam"], state)
    assert torch.equal(state, out) and torch.equal(y2, y)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_steps_continue_a_prefill(dev, dtype):
    """Prefill, then tokens one by one, against the whole in one."""
    lens, d = [37, 150, 5], 96
    c, n = make(dev, lens, d, dtype, False)
    want = ref.Recurrence(n["x"], n["rg"], n["ig"], n["lam"], n["cu"], 8.0, None)
    keep = [ln - 4 for ln in lens]
    rows = np.concatenate([np.arange(lo, lo + k) for lo, k in zip(n["cu"], keep)])
    cut = torch.from_numpy(rows).to(dev)
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(keep)]).astype(np.int32)).to(dev)
    y, state = ops.gated_recurrence(*(c[k][cut] for k in ("x", "rg", "ig")), c["lam"], cu)
    near(y, want.h[rows], want.eh[rows], dtype, "prefill")
    for i in range(4):
        at = n["cu"][:-1] + np.array(keep) + i
        idx = torch.from_numpy(at.astype(np.int64)).to(dev)
        y = ops.gated_recurrence_step(*(c[k][idx] for k in ("x", "rg", "ig")), c["lam"], state)
        near(y, want.h[at], want.eh[at], dtype, f"token {i}")


def test_streams_and_graphs(dev):
    """Captured and replayed among eager calls of other sizes; two streams at once."""
    c, _ = make(dev, [700, 0, 900], 200, "bf16", True)
    o, _ = make(dev, [3000], 64, "bf16", False)

    def both():
        y, final, carry = forward(c)
        return [y, final, *backward(c, carry).values()]

    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        side = [both() for _ in range(3)]
    here = [both() for _ in range(3)]
    torch.cuda.synchronize()
    for r in side + here:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            out = both()
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(4):
        for t in out:
            t.fill_(float("nan"))
        backward(o, forward(o)[2])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_full_cards_at_once(dev):
    """Calls that could each fill the card, on two streams: their workgroups wait for started ones only."""
    torch.manual_seed(8)
    t, d = 20011, 1024
    sets = []
    for i in range(2):
        c = {k: torch.randn((t, d), device=dev).to(torch.bfloat16) for k in ("x", "rg", "ig", "dy")}
        c["lam"] = torch.randn(d, device=dev) - 4.0
        c["cu"] = torch.tensor([0, 9000 + i, 9000 + i, t - 5 * i], dtype=torch.int32, device=dev)
        c["h0"], c["dfinal"] = (torch.randn((3, d), device=dev) for _ in range(2))
        sets.append(c)

    def both(c):
        y, final, carry = forward(c)
        return [y, final, *backward(c, carry).values()]

    want = [both(c) for c in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, both(sets[i])))
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lam", [-5.0, 0.0, 4.0])
def test_nan_reaches_the_end(dev, dtype, lam):
    """What is not a number stays one to the end of its sequence (backwards: to its start), however strong
    the decays are, in its own channel and sequence only."""
    torch.manual_seed(9)
    d, cu = 70, [0, 300, 5000, 5200]
    c = {k: torch.randn((5200, d), device=dev).to(DT[dtype]) for k in ("x", "rg", "ig", "dy")}
    c["lam"] = torch.full((d,), lam, device=dev)
    c["cu"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    c["h0"], c["dfinal"] = (torch.randn((3, d), device=dev) for _ in range(2))
    c["x"][310, 5] = float("nan")
    c["dy"][4990, 7] = float("nan")
    y, final, carry = forward(c)
    want = torch.zeros(5200, d, dtype=torch.bool, device=dev)
    want[310:5000, 5] = True
    assert torch.equal(y.isnan(), want) and final.isnan().nonzero().tolist() == [[1, 5]]
    g = backward(c, carry)
    # (the channel of the missing x: what lies before it has a gradient; its own x has none that meets it)
    back = torch.zeros(5200, d, dtype=torch.bool, device=dev)
    back[300:4991, 7] = True
    assert torch.equal(g["dx"].isnan(), back)
    assert g["dinitial"].isnan().nonzero().tolist() == [[1, 7]]
    assert g["dlam"].isnan().nonzero().flatten().tolist() == [5, 7]
