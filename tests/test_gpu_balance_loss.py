"""The router's balance loss, counts and gradient against float64: batches and ragged sequences,
padding rows, choices of no expert, odd widths, strided logits, captured calls."""
import numpy as np
import pytest
import torch

import train_ref as ref
from reimagined_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(dev, rows, e, k, dtype, pad, lens, seed=0):
    rng = np.random.default_rng([rows, e, k, seed])
    t = torch.from_numpy((1.5 * rng.standard_normal((rows, e)) + 0.5 * rng.standard_normal(e))
                         .astype(np.float32)).to(DT[dtype])
    x = t.double().numpy()
    sel = np.argsort(-x, axis=1, kind="stable")[:, :k].astype(np.int32)
    valid = None
    if pad:
        valid = (rng.random(rows) > 0.25).astype(np.uint8)
        sel[valid == 0] = -1
        if rows > 3:
            sel[3, 0] = -1  # a valid row that names one expert less
    cu = None if lens is None else np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    g = lambda a: None if a is None else torch.from_numpy(a).to(dev)
    return t.to(dev), x, g(sel), sel, g(valid), valid, g(cu), cu


def near(got, want, lim, what):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= lim + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / (lim + 1e-37))))


def check(dev, rows, e, k, dtype, score, pad, lens):
    t, x, sel_t, sel, valid_t, valid, cu_t, cu = make(dev, rows, e, k, dtype, pad, lens)
    f = ops.moe_balance_loss(t, sel_t, score=score, cu_seqlens=cu_t, valid_rows=valid_t)
    loss, counts, tokens, mean, dx, lim = ref.balance(x, sel, score, cu, valid, 0.5)
    assert np.array_equal(f["counts"].cpu().numpy(), counts)
    assert np.array_equal(f["tokens"].cpu().numpy(), tokens)
    # a probability is off by 2 U a unit of the exponent and 80 U; the rows' sums by their depth
    reach = np.abs(x).max() * 2 + 1
    rel = (2 * reach + 80 + 64 + rows / 256) * ref.U
    near(f["mean_prob"], mean, rel * mean, "mean_prob")
    near(f["loss"], np.array([loss]), np.array([(rel + 4 * ref.U) * loss]), "loss")
    scale = torch.tensor([0.5], device=dev)
    for dloss in (0.5, scale):
        d = ops.moe_balance_loss_backward(t, f["counts"], f["tokens"], k, score=score, cu_seqlens=cu_t,
                                          valid_rows=valid_t, dloss=dloss)
        assert d.dtype == t.dtype
        near(d, dx, lim + ref.HALF_STEP[dtype] * np.abs(dx) * (1 + 2.0**-7), "dlogits")
    g = ops.moe_balance_loss(t, sel_t, score=score, cu_seqlens=cu_t, valid_rows=valid_t)
    assert all(torch.equal(f[n], g[n]) for n in f)
    return f


@pytest.mark.parametrize("rows,e,k", [(1, 1, 1), (1, 8, 2), (127, 16, 1), (128, 17, 3), (129, 33, 4), (300, 60, 6),
                                      (1000, 64, 16), (77, 129, 8), (2049, 256, 8), (515, 300, 2), (260, 512, 16)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("pad", [False, True])
def test_batch(dev, rows, e, k, dtype, score, pad):
    check(dev, rows, e, k, dtype, score, pad, None)


@pytest.mark.parametrize("lens", [[5], [0, 7, 0], [128, 128], [127, 1, 130, 0, 0, 62], [1] * 200, [2] * 1500,
                                  [0] * 1100 + [90, 300], [1000, 3]], ids=lambda v: f"{len(v)}x{sum(v)}")
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("pad", [False, True])
def test_sequences(dev, lens, score, pad):
    check(dev, sum(lens), 24, 3, "f32", score, pad, lens)
    check(dev, sum(lens), 70, 2, "bf16", score, pad, lens)


def test_padding_reaches_nothing(dev):
    """Padding rows, and rows of no sequence, hold NaN; a sequence has no valid row."""
    rows, e, k = 400, 40, 4
    t, x, sel_t, sel, _, _, _, _ = make(dev, rows, e, k, "f32", False, None)
    valid = np.ones(rows, np.uint8)
    valid[100:150] = 0
    valid[::9] = 0
    cu = torch.tensor([20, 100, 150, 380], dtype=torch.int32, device=dev)
    bad = t.clone()
    out = torch.from_numpy(valid == 0).to(dev)
    out[:20] = True
    out[380:] = True
    bad[out] = float("nan")
    vt = torch.from_numpy(valid).to(dev)
    f = ops.moe_balance_loss(bad, sel_t, cu_seqlens=cu, valid_rows=vt)
    want = ref.balance(x, sel, "softmax", [20, 100, 150, 380], valid, 1.0)
    assert f["tokens"][1] == 0 and not f["counts"][1].any() and not f["mean_prob"][1].any()
    assert np.array_equal(f["counts"].cpu().numpy(), want[1])
    near(f["loss"], np.array([want[0]]), np.array([200 * ref.U * want[0]]), "loss")
    d = ops.moe_balance_loss_backward(bad, f["counts"], f["tokens"], k, cu_seqlens=cu, valid_rows=vt)
    assert not d[out].any()
    near(d, want[4], want[5] + ref.U * np.abs(want[4]), "dlogits")
    none = ops.moe_balance_loss(bad, sel_t, valid_rows=torch.zeros(rows, dtype=torch.uint8, device=dev))
    assert none["loss"] == 0 and not none["counts"].any() and not none["mean_prob"].any()
    d = ops.moe_balance_loss_backward(bad, none["counts"], none["tokens"], k,
                                      valid_rows=torch.zeros(rows, dtype=torch.uint8, device=dev))
    assert not d.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("e", [5, 64, 131])
def test_strided_and_added(dev, dtype, e):
    """Logits as a column slice at an odd offset, masked experts at -inf; the gradient on top of
    another one, also in place."""
    rows, k = 150, 2
    t, *_ = make(dev, rows, e, k, dtype, False, None)
    t[:, 1] = float("-inf")
    sel = t.float().sort(dim=1, descending=True, stable=True).indices[:, :k].int().contiguous()
    wide = torch.full((rows, e + 3), float("nan"), dtype=DT[dtype], device=dev)
    view = wide[:, 1:1 + e]
    view.copy_(t)
    f, g = ops.moe_balance_loss(t, sel), ops.moe_balance_loss(view, sel)
    assert all(torch.equal(f[n], g[n]) for n in f) and torch.isfinite(f["loss"]).all()
    assert f["mean_prob"][0, 1] == 0
    d = ops.moe_balance_loss_backward(t, f["counts"], f["tokens"], k)
    assert not d[:, 1].any() and torch.isfinite(d).all()
    assert torch.equal(d, ops.moe_balance_loss_backward(view, f["counts"], f["tokens"], k))
    add = torch.randn((rows, e), device=dev).to(DT[dtype])
    got = ops.moe_balance_loss_backward(t, f["counts"], f["tokens"], k, dloss=3.0, add=add)
    exact = ops.moe_balance_loss_backward(t.float(), f["counts"], f["tokens"], k, dloss=3.0)
    want = exact.double() + add.double()
    lim = ref.HALF_STEP[dtype] * want.abs() * (1 + 2.0**-7) + 4 * ref.U * exact.double().abs()
    assert ((got.double() - want).abs() <= lim).all()


def test_behind_the_router(dev):
    """On the router's own choices: the counts are its counts, the loss of a uniform router is 1."""
    rows, e, k = 1024, 32, 4
    logits = torch.randn((rows, e), device=dev)
    r = ops.moe_route_scored(logits, k, score="sigmoid")
    f = ops.moe_balance_loss(logits, r["selected"], score="sigmoid")
    assert torch.equal(f["counts"][0], r["counts"]) and f["tokens"].item() == rows
    even = torch.zeros((rows, e), device=dev)
    sel = (torch.arange(rows * k, device=dev) % e).view(rows, k).int()
    f = ops.moe_balance_loss(even, sel)
    assert abs(f["loss"].item() - 1.0) <= 100 * ref.U
    d = ops.moe_balance_loss_backward(even, f["counts"], f["tokens"], k)
    # every count is rows k / e: the gradient is the rounding of count - sum count p
    assert d.abs().max().item() <= 100 * ref.U * e / rows


def test_streams_and_graphs(dev):
    lens = [300, 0, 700, 24]
    t, _, sel, _, valid, _, cu, _ = make(dev, sum(lens), 60, 4, "f32", True, lens)

    def both():
        f = ops.moe_balance_loss(t, sel, cu_seqlens=cu, valid_rows=valid)
        return [*f.values(), ops.moe_balance_loss_backward(t, f["counts"], f["tokens"], 4, cu_seqlens=cu,
                                                           valid_rows=valid)]

    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        side = both()
        with torch.cuda.graph(g, stream=s):
            out = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, want))
    for _ in range(3):
        for a in out:
            a.fill_(7)
        ops.moe_balance_loss(torch.randn((5000, 200), device=dev),
                             torch.zeros((5000, 3), dtype=torch.int32, device=dev))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e", [3, 24, 200])
def test_far_logits(dev, dtype, score, e):
    """Rows far below 0, whose sigmoids a float cannot hold, and experts masked by the type's lowest value."""
    rng = np.random.default_rng(e)
    rows, k = 150, 2
    x = 2.0 * rng.standard_normal((rows, e)) + np.array([0.0, -55.0, -62.0, -88.0, -300.0, 80.0])[np.arange(rows) % 6, None]
    t = torch.from_numpy(x.astype(np.float32)).to(DT[dtype])
    t[::7, 1] = torch.finfo(DT[dtype]).min
    x = t.double().numpy()
    sel = np.argsort(-x, axis=1, kind="stable")[:, :k].astype(np.int32)
    t, sel_t = t.to(dev), torch.from_numpy(sel).to(dev)
    f = ops.moe_balance_loss(t, sel_t, score=score)
    loss, counts, _, mean, dx, lim = ref.balance(x, sel, score, None, None, 1.0)
    assert np.array_equal(f["counts"].cpu().numpy(), counts)
    # (as above; what is masked adds nothing, and of a row only the largest matter: 320 at most)
    rel = (2 * 321 + 80 + 64 + 1) * ref.U
    near(f["mean_prob"], mean, rel * mean, "mean_prob")
    near(f["loss"], np.array([loss]), np.array([(rel + 4 * ref.U) * loss]), "loss")
    d = ops.moe_balance_loss_backward(t, f["counts"], f["tokens"], k, score=score)
    near(d, dx, lim + ref.HALF_STEP[dtype] * np.abs(dx) * (1 + 2.0**-7), "dlogits")


@pytest.mark.parametrize("lens", [None, [30000, 0, 33, 100] + [1] * 200 + [39700], [10] * 6500 + [7], [70001]],
                         ids=["batch", "mixed", "many", "one"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("pad", [False, True])
def test_many_rows(dev, lens, score, pad):
    """Blocks of several steps, borders inside and between them, loss parts in the thousands."""
    rows = 70001 if lens is None else sum(lens)
    check(dev, rows, 20, 2, "f32", score, pad, lens)
    check(dev, rows, 37, 3, "bf16", score, pad, lens)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,k", [(4, 4), (7, 7), (48, 3)])
def test_balanced(dev, dtype, score, e, k):
    """Experts that all have the same load: the gradient is 0, not what rounding leaves of it; and one choice
    more of one of them shows with all of its bits."""
    rows = 48 * 20
    x = torch.randn((rows, e), device=dev, generator=torch.Generator(dev).manual_seed(e)).to(DT[dtype])
    sel = torch.stack([(torch.arange(rows, device=dev) + i * (e // k)) % e for i in range(k)], 1).int()
    rows = rows if k < e else 7
    x, sel = x[:rows], sel[:rows].contiguous()
    f = ops.moe_balance_loss(x, sel, score=score)
    assert (f["counts"] == rows * k // e).all()
    back = lambda counts: ops.moe_balance_loss_backward(x, counts, f["tokens"], k, score=score)
    assert not back(f["counts"]).any()
    counts = f["counts"].clone()
    counts[0, 1] += 1
    xd = x.double()
    p = torch.softmax(xd, 1) if score == "softmax" else torch.sigmoid(xd) / torch.sigmoid(xd).sum(1, keepdim=True)
    one = torch.zeros(e, device=dev, dtype=torch.float64)
    one[1] = 1.0
    want = e / (k * float(rows) ** 2) * p * (one - p[:, 1:2])
    if score == "sigmoid":
        want = want * torch.sigmoid(-xd)
    # a probability is off by 2 U a unit of the exponent (10 at most here) and 80 U, twice; twelve roundings
    lim = e / (k * float(rows) ** 2) * p * (one + p[:, 1:2]) * (2 * (2 * 10 + 80) + 12) * ref.U
    near(back(counts), want.cpu().numpy(), (lim + ref.HALF_STEP[dtype] * want.abs() * (1 + 2.0**-7)).cpu().numpy(), "dlogits")
