"""Scored expert routing and its gradient against the definition in 64 bits: scores, bias,
groups, ties, unavailable experts, padding rows, the dispatch, and the gradient against its
formula and against differences."""
import numpy as np
import pytest
import torch

from reimagined_amd import ops

pytestmark = pytest.mark.gpu


def scores64(x, score):
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return 1.0 / (1.0 + np.exp(-x))
    with np.errstate(invalid="ignore"):
        e = np.exp(x - x.max(1, keepdims=True))
    e[np.isneginf(x)] = 0.0
    return e / np.where(e.sum(1, keepdims=True) > 0, e.sum(1, keepdims=True), 1.0)


def route64(x, k, score, bias=None, groups=1, keep=1, best=2, renorm=True, scale=1.0, valid=None):
    """The definition, row by row, in 64 bits -> weights, selected."""
    rows, e = x.shape
    s = scores64(x, score)
    c = s + (0.0 if bias is None else bias[None].astype(np.float64))
    if bias is None and (groups == 1 or best == 1):
        c = x.copy()
    c[np.isneginf(x)] = -np.inf
    w = np.zeros((rows, k))
    sel = np.full((rows, k), -1, np.int64)
    for r in range(rows):
        if valid is not None and not valid[r]:
            continue
        row = c[r].copy()
        if groups > 1 and keep < groups:
            size = e // groups
            gs = []
            for g in range(groups):
                top = np.sort(row[g * size:(g + 1) * size])[::-1][:best]
                top = top[~np.isneginf(top)]
                gs.append(top.sum() if len(top) else -np.inf)
            order = np.argsort(-np.array(gs), kind="stable")[:keep]
            for g in range(groups):
                if g not in order:
                    row[g * size:(g + 1) * size] = -np.inf
        pick = [i for i in np.argsort(-row, kind="stable")[:k] if not np.isneginf(row[i])]
        sel[r, :len(pick)] = pick
        if not pick:
            continue
        if renorm:  # a softmax over the choice (of the logits, or of the sigmoids' logarithms)
            l = x[r, pick] if score == "softmax" else -np.logaddexp(0.0, -x[r, pick])
            t = np.exp(l - l.max())
            w[r, :len(pick)] = t / t.sum() * scale
        else:
            w[r, :len(pick)] = s[r, pick] * scale
    return w, sel


def dispatch_ref(sel, e):
    rows, k = sel.shape
    counts = np.bincount(sel[sel >= 0], minlength=e)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    perm = np.full(rows * k, -1)
    slot_of = np.full((rows, k), -1)
    at = offsets[:-1].copy()
    for r in range(rows):
        for i in range(k):
            if sel[r, i] >= 0:
                slot_of[r, i] = at[sel[r, i]]
                perm[at[sel[r, i]]] = r
                at[sel[r, i]] += 1
    return counts, offsets, perm, slot_of


def rtol(x):
    """A weight is a quotient of at most E + 16 exponentials' sum: half a step for each sum
    (36 additions on the longest path: 32 in a lane, 4 across lanes), two steps for each
    exponential and quotient (32 for all of them together), and the rounding of the difference that the
    exponential takes, at most the logits' range (a mask's lowest value gives exact zeros), for
    numerator and denominator."""
    f = x[np.abs(x) < 1e30]
    span = float(f.max() - f.min()) if f.size else 0.0
    return (36 + 32 + 2 * span) * 2.0**-24


def check(dev, x, k, dtype=torch.float32, **kw):
    xt = torch.from_numpy(x.astype(np.float32)).to(dtype)
    x64 = xt.double().numpy()
    bias, valid = kw.pop("bias", None), kw.pop("valid", None)
    want_w, want_sel = route64(x64, k, kw.get("score", "softmax"), bias, kw.get("groups", 1),
                               kw.get("group_keep", kw.get("groups", 1)), kw.get("group_best", 2),
                               kw.get("renorm", True), kw.get("scale", 1.0), valid)
    bt = None if bias is None else torch.from_numpy(bias).to(dev)
    vt = None if valid is None else torch.from_numpy(valid).to(dev)
    r = ops.moe_route_scored(xt.to(dev), k, bias=bt, valid_rows=vt, **kw)
    only = ops.moe_route_scored(xt.to(dev), k, bias=bt, valid_rows=vt, select_only=True, **kw)
    got = {n: v.cpu().numpy() for n, v in r.items()}
    np.testing.assert_array_equal(got["selected"], want_sel)
    for n, want in zip(("counts", "offsets", "perm", "slot_of"), dispatch_ref(want_sel, x.shape[1])):
        np.testing.assert_array_equal(got[n], want, err_msg=n)
    np.testing.assert_allclose(got["weights"], want_w, rtol=rtol(x64), atol=1e-37)
    assert set(only) == {"weights", "selected"}
    assert torch.equal(only["weights"], r["weights"])
    assert torch.equal(only["selected"], r["selected"])
    return r


@pytest.mark.parametrize("rows,e,k", [(1, 1, 1), (1, 64, 6), (7, 3, 3), (16, 8, 2), (33, 17, 5),
                                      (64, 256, 8), (65, 60, 4), (257, 33, 16), (300, 512, 10),
                                      (4097, 100, 3), (5000, 256, 8), (8200, 64, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_sizes(dev, rows, e, k, score, biased):
    rng = np.random.default_rng([rows, e, k, biased])
    x = rng.normal(0, 1.5, (rows, e))
    bias = rng.normal(0, 0.1, e).astype(np.float32) if biased else None
    check(dev, x, k, score=score, bias=bias, renorm=rows % 2 == 0, scale=2.5,
          dtype=torch.bfloat16 if e % 3 == 0 else torch.float32)


@pytest.mark.parametrize("e,groups,keep", [(256, 8, 4), (60, 4, 2), (48, 16, 5), (160, 8, 3),
                                           (512, 16, 1), (30, 2, 1), (16, 16, 3), (8, 4, 4)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("biased", [False, True])
def test_groups(dev, e, groups, keep, best, biased):
    rng = np.random.default_rng([e, groups, keep, best])
    x = rng.normal(0, 1.5, (211, e))
    bias = rng.normal(0, 0.2, e).astype(np.float32) if biased else None
    k = min(3, keep * (e // groups))
    for score in ("softmax", "sigmoid"):
        check(dev, x, k, score=score, bias=bias, groups=groups, group_keep=keep, group_best=best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_ties_go_to_the_lower_index(dev, score, groups):
    rng = np.random.default_rng(5)
    x = rng.integers(-2, 3, (130, 64)).astype(np.float32)
    x[0] = 0.0
    kw = dict(score=score, groups=groups, group_keep=min(groups, 2))
    check(dev, x, 7, **kw)
    check(dev, x, 7, dtype=torch.bfloat16, **kw)
    # equal logits and steps of the bias: sums that are equal in 64 bits
    check(dev, x, 7, bias=(rng.integers(0, 3, 64) * 0.25).astype(np.float32), **kw)
    check(dev, x, 7, bias=np.zeros(64, np.float32), **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_values_next_to_each_other(dev, score):
    """Logits one float apart, and biases that bring distant scores within 1e-9 of each other:
    32-bit scores cannot tell them apart, the choice has to."""
    rng = np.random.default_rng(6)
    e = 40
    x = np.float32(1.0) + rng.permuted(np.tile(np.arange(e), (90, 1)), axis=1) * np.float32(2.0**-23)
    x = x.astype(np.float32)
    check(dev, x, 9, score=score)
    check(dev, x, 9, score=score, bias=np.full(e, 0.125, np.float32))
    y = rng.normal(0, 1, (1, e)).astype(np.float32).repeat(50, 0)
    s = scores64(y[:1].astype(np.float64), score)[0]
    bias = (0.5 - s).astype(np.float32)  # every sum within 2^-25 of 0.5
    check(dev, y, 9, score=score, bias=bias)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
def test_unavailable_experts(dev, score, biased, groups, keep):
    """-inf logits: fewer than k experts, a whole group, a row with none; and masks of the type's
    lowest value, which stay finite."""
    rng = np.random.default_rng(7)
    x = rng.normal(0, 1, (40, 32)).astype(np.float32)
    x[0, 2:] = -np.inf
    x[1] = -np.inf
    x[2, 8:16] = -np.inf
    x[3, 1:] = np.finfo(np.float32).min
    x[4] = np.finfo(np.float32).min
    x[5, ::2] = -np.inf
    x[6, 31:] = -np.inf
    bias = rng.normal(0, 0.1, 32).astype(np.float32) if biased else None
    for renorm in (True, False):
        check(dev, x, 5, score=score, bias=bias, groups=groups, group_keep=keep, renorm=renorm)
    if biased:
        bias[3] = -np.inf
        want = ops.moe_route_scored(torch.from_numpy(x).to(dev), 5, score=score,
                                    bias=torch.from_numpy(bias).to(dev))["selected"]
        assert not (want == 3).any()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_extreme_logits(dev, score):
    """Scores that underflow: the renormalised weights are those of the choice."""
    rng = np.random.default_rng(8)
    x = rng.normal(0, 1, (20, 16)).astype(np.float32)
    x[:10] -= 300.0
    x[10:15] += 300.0
    check(dev, x, 4, score=score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_nan_rows(dev, score, biased):
    rng = np.random.default_rng(9)
    x = rng.normal(0, 1, (70, 24)).astype(np.float32)
    x[3, 5] = np.nan
    x[66, 23] = np.nan
    bias = torch.zeros(24, device=dev) if biased else None
    r = ops.moe_route_scored(torch.from_numpy(x).to(dev), 3, score=score, bias=bias)
    sel, w = r["selected"].cpu().numpy(), r["weights"].cpu().numpy()
    for row in (3, 66):
        assert sel[row].tolist() == [0, 1, 2] and np.isnan(w[row]).all()
    good = [i for i in range(70) if i not in (3, 66)]
    want_w, want_sel = route64(x[good].astype(np.float64), 3, score,
                               np.zeros(24, np.float32) if biased else None)
    np.testing.assert_array_equal(sel[good], want_sel)
    np.testing.assert_allclose(w[good], want_w, rtol=rtol(x[good]))
    counts, offsets, perm, slot_of = dispatch_ref(sel, 24)
    np.testing.assert_array_equal(r["perm"].cpu().numpy(), perm)


@pytest.mark.parametrize("rows", [1, 30, 500, 9000])
def test_padding_rows(dev, rows):
    rng = np.random.default_rng(rows)
    x = rng.normal(0, 1.5, (rows, 48))
    valid = (rng.random(rows) < 0.7).astype(np.uint8)
    check(dev, x, 4, score="sigmoid", valid=valid, bias=rng.normal(0, 0.1, 48).astype(np.float32))
    check(dev, x, 4, valid=np.zeros(rows, np.uint8))


def test_strided_logits(dev):
    rng = np.random.default_rng(11)
    wide = torch.from_numpy(rng.normal(0, 1, (77, 100)).astype(np.float32)).to(dev)
    part = wide[:, 13:13 + 40]
    a = ops.moe_route_scored(part, 4, score="sigmoid")
    b = ops.moe_route_scored(part.contiguous(), 4, score="sigmoid")
    assert all(torch.equal(a[n], b[n]) for n in b)
    g = torch.randn(77, 4, device=dev)
    for renorm in (True, False):
        assert torch.equal(
            ops.moe_route_scored_backward(part, a["selected"], g, renorm=renorm),
            ops.moe_route_scored_backward(part.contiguous(), a["selected"], g, renorm=renorm))


# ---- gradient -----------------------------------------------------------------------

def weights64(x, sel, score, renorm, scale):
    """Weights of a given choice (sel [rows, k], all >= 0), in 64 bits."""
    s = scores64(x, score)
    w = np.take_along_axis(s, sel, 1)
    return (w / w.sum(1, keepdims=True) if renorm else w) * scale


def grad64(x, sel, g, score, renorm, scale):
    s = scores64(x, score)
    g = np.where(sel < 0, 0.0, g) * scale
    out = np.zeros_like(x)
    for r in range(len(x)):
        on = sel[r] >= 0
        at = sel[r][on]
        t = s[r, at]
        ds = g[r][on].copy()
        if renorm and len(at):
            ds = (ds - (ds * t).sum() / t.sum()) / t.sum()
        full = np.zeros(x.shape[1])
        np.add.at(full, at, ds)
        out[r] = full * s[r] * (1 - s[r]) if score == "sigmoid" else s[r] * (full - full @ s[r])
    return out


@pytest.mark.parametrize("rows,e,k", [(1, 1, 1), (5, 4, 4), (17, 60, 4), (100, 256, 8), (33, 512, 16),
                                      (1000, 64, 6)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient(dev, rows, e, k, score, renorm, dtype):
    rng = np.random.default_rng([rows, e, k])
    xt = torch.from_numpy(rng.normal(0, 1.5, (rows, e)).astype(np.float32)).to(dtype)
    x = xt.double().numpy()
    sel = ops.moe_route_scored(xt.to(dev), k, score=score, renorm=renorm)["selected"]
    sel_n = sel.cpu().numpy().astype(np.int64)
    g = rng.normal(0, 1, (rows, k)).astype(np.float32)
    got = ops.moe_route_scored_backward(xt.to(dev), sel, torch.from_numpy(g).to(dev), score=score,
                                        renorm=renorm, scale=2.5)
    assert got.dtype == dtype
    got = got.double().cpu().numpy()
    want = grad64(x, sel_n, g.astype(np.float64), score, renorm, 2.5)
    # every score is off by rtol() of itself, the sum over the choice has 16 terms, and each
    # product one rounding more: all against the row's largest |g| * scale, of which a gradient
    # is at most a weighted mean
    atol = 2 * (rtol(x) + 24 * 2.0**-24) * 2.5 * np.abs(g).max(1, keepdims=True)
    lim = atol + torch.finfo(dtype).eps / 2 * np.abs(want)
    assert (np.abs(got - want) <= lim).all(), np.abs(got - want).max()
    if dtype == torch.float32 and rows <= 17:
        h = 1e-4  # central differences: h^2 * the third derivative (below 1) off
        for j in range(e):
            up, dn = x.copy(), x.copy()
            up[:, j] += h
            dn[:, j] -= h
            d = (weights64(up, sel_n, score, renorm, 2.5) - weights64(dn, sel_n, score, renorm, 2.5))
            num = (d / (2 * h) * g).sum(1)
            err = np.abs(got[:, j] - num)
            assert (err <= atol[:, 0] + k * 2.5 * h * h * np.abs(g).max(1)).all()


def test_gradient_of_padding_and_repeated_choices(dev):
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (20, 12)).astype(np.float32)
    sel = np.stack([rng.permutation(12)[:4] for _ in range(20)])
    sel[2] = -1
    sel[5, 2:] = -1
    sel[7] = [3, 3, 1, 3]  # one expert named three times: the gradients add
    g = rng.normal(0, 1, (20, 4)).astype(np.float32)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            got = ops.moe_route_scored_backward(
                torch.from_numpy(x).to(dev), torch.from_numpy(sel.astype(np.int32)).to(dev),
                torch.from_numpy(g).to(dev), score=score, renorm=renorm).cpu().numpy()
            want = grad64(x.astype(np.float64), sel, g.astype(np.float64), score, renorm, 1.0)
            atol = 6 * (rtol(x) + 24 * 2.0**-24) * np.abs(g).max(1, keepdims=True)
            assert (np.abs(got - want) <= atol).all()
            assert (got[2] == 0).all()


def test_gradient_ignores_unavailable_experts(dev):
    x = torch.zeros(3, 6, device=dev)
    x[1, 2:] = -torch.inf
    x[2] = -torch.inf
    r = ops.moe_route_scored(x, 3, renorm=False)
    assert r["selected"][1].tolist() == [0, 1, -1] and r["selected"][2].tolist() == [-1] * 3
    for renorm in (True, False):
        for score in ("softmax", "sigmoid"):
            g = ops.moe_route_scored_backward(x, r["selected"], torch.ones(3, 3, device=dev),
                                              score=score, renorm=renorm)
            assert torch.isfinite(g).all() and (g[1, 2:] == 0).all() and (g[2] == 0).all()


@pytest.mark.parametrize("e,groups,keep", [(504, 9, 4), (495, 15, 2), (330, 3, 2), (320, 5, 4), (252, 12, 5),
                                           (9, 3, 2), (64, 2, 1), (512, 2, 1), (40, 8, 3), (144, 16, 7), (56, 2, 1), (112, 4, 3),
                                           (24, 2, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_layouts(dev, e, groups, keep, dtype):
    """Groups over every number of lanes, and more experts of a group than its lanes hold."""
    rng = np.random.default_rng([e, groups])
    for rows in (3, 70, 333):
        x = rng.normal(0, 1.5, (rows, e))
        bias = rng.normal(0, 0.1, e).astype(np.float32)
        for best in (1, 2):
            for b in (None, bias):
                check(dev, x, min(4, keep * (e // groups)), dtype=dtype, score="softmax" if best == 1 else "sigmoid",
                      bias=b, groups=groups, group_keep=keep, group_best=best)


@pytest.mark.parametrize("e,k,groups", [(64, 8, 1), (256, 8, 8), (256, 15, 1), (256, 16, 1), (512, 5, 4),
                                        (40, 1, 1), (24, 11, 2)])
@pytest.mark.parametrize("near", ["choices", "one more", "two more"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_only_the_choices_lie_together(dev, e, k, groups, near, score):
    """The k largest values (and one, or two, behind them) within 2^-24 of each other in an order that
    32 bits do not show, all others far below: of logits, and of scores with a bias."""
    rng = np.random.default_rng([e, k, groups])
    rows, half = 131, e // 2 if groups > 1 else e  # (the near ones in the groups that stay)
    count = min(k + {"choices": 0, "one more": 1, "two more": 2}[near], half)
    kw = dict(score=score, groups=groups, group_keep=max(groups // 2, 1))
    x = rng.uniform(-3, -2, (rows, e))
    for r in range(rows):
        at = rng.permutation(half)[:count]
        x[r, at] = 1.0 + rng.permutation(count) % 5 * 2.0**-23
        if groups > 1:  # and a value in each of those groups that keeps them clear of the others
            size = e // groups
            for g in range(groups // 2):
                x[r, g * size:g * size + 2] = np.maximum(x[r, g * size:g * size + 2], 0.5 + 0.01 * g)
    x = x.astype(np.float32)
    check(dev, x, k, **kw)
    # sums with a bias: each row's near experts get the same place by their own logits
    y = x[:1].repeat(rows, 0)
    s = scores64(y[:1].astype(np.float64), score)[0]
    bias = np.where(x[0] >= 1.0, 0.9 - s, -0.05).astype(np.float32)
    check(dev, y, k, bias=bias, **kw)


@pytest.mark.parametrize("rows,e,k", [(16384, 256, 8), (16500, 256, 3), (65535, 4, 1), (65536, 4, 1),
                                      (65535, 5, 3), (8192, 509, 2), (3000, 6, 6)])
def test_counts_of_blocks(dev, rows, e, k):
    """Around what the counts' bytes and pairs hold, an expert that every row takes among them."""
    rng = np.random.default_rng([rows, e])
    x = rng.normal(0, 1, (rows, e))
    x[:, e // 2] = 9.0
    r = ops.moe_route_scored(torch.from_numpy(x.astype(np.float32)).to(dev), k)
    got = {n: v.cpu().numpy() for n, v in r.items()}
    want = np.argsort(-x.astype(np.float32), axis=1, kind="stable")[:, :k]
    np.testing.assert_array_equal(got["selected"], want)
    counts = np.bincount(want.ravel(), minlength=e)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    # slots: expert-major, rows ascending
    perm = np.argsort(want.ravel(), kind="stable")
    slot_of = np.empty(rows * k, np.int64)
    slot_of[perm] = np.arange(rows * k)
    for n, v in (("counts", counts), ("offsets", offsets), ("perm", perm // k),
                 ("slot_of", slot_of.reshape(rows, k))):
        np.testing.assert_array_equal(got[n], v, err_msg=n)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups", [(24, 1), (24, 4), (256, 8), (300, 1)])
def test_infinite_biases(dev, score, e, groups):
    """-inf takes an expert out for every row, +inf puts one first, also where a logit is -inf."""
    rng = np.random.default_rng([e, groups])
    x = rng.normal(0, 1, (70, e)).astype(np.float32)
    x[::3, 5] = x[1::4, 7] = -np.inf
    bias = rng.normal(0, 0.1, e).astype(np.float32)
    bias[2] = bias[7] = -np.inf
    kw = dict(score=score, groups=groups, group_keep=max(groups // 2, 1))
    check(dev, x, 4, bias=bias, **kw)
    bias[5] = np.inf
    check(dev, x, 4, bias=bias, **kw)


@pytest.mark.parametrize("mask", [-20.0, -100.0, -1e3, -1e4, -1e5, 1e4])
@pytest.mark.parametrize("usable", [1, 2])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_groups_behind_large_finite_biases(dev, mask, usable, score, renorm):
    """A mask that stays finite on all but `usable` experts of a group: with one, a group's score holds
    the mask, and its step in 32 bits is far above that of the scores.  The groups' sums lie
    within a few such steps of each other, in an order that only 64 bits show."""
    rng = np.random.default_rng([int(abs(mask)), usable, score == "softmax"])
    rows, groups, size = 400, 4, 4
    step = float(np.spacing(np.float32(abs(mask))))
    s = rng.uniform(0.02, 0.03, (rows, groups, size))
    s[:, :, 0] = rng.uniform(0.3, 0.6, (rows, groups))
    s[:, :, 1] = np.clip(0.9 - s[:, :, 0] + rng.uniform(-2, 2, (rows, groups)) * step, 1e-3, 0.95)
    s = s.reshape(rows, -1)
    x = (np.log(s) if score == "softmax" else np.log(s / (1 - s))).astype(np.float32)
    bias = np.zeros((groups, size), np.float32)
    bias[:, usable:] = mask
    check(dev, x, 2, score=score, bias=bias.ravel(), groups=groups, group_keep=2, renorm=renorm, scale=2.5)


def test_groups_of_two_masks(dev):
    """Sums of -9999.173378 and -9999.173233, which rounding to 32 bits puts in the other order."""
    x = np.array([[-0.50692, -0.19781, 0.52821, -1.40072]], np.float32)
    check(dev, x, 1, score="sigmoid", bias=np.array([0, -1e4, 0, -1e4], np.float32), groups=2, group_keep=1)


@pytest.mark.parametrize("mask", [-1e3, -1e5, float(np.finfo(np.float32).min)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_masked_whole(dev, mask, score):
    """Groups without a usable expert beside groups with one, two and all of them."""
    rng = np.random.default_rng(13)
    x = rng.normal(0, 1.5, (300, 48)).astype(np.float32)
    bias = rng.normal(0, 0.1, (6, 8)).astype(np.float32)
    bias[0] = bias[1, 1:] = bias[3, 2:] = mask
    check(dev, x, 3, score=score, bias=bias.ravel(), groups=6, group_keep=3)


@pytest.mark.parametrize("e,k", [(12, 4), (256, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_padding_rows_that_hold_anything(dev, e, k, score, renorm, dtype):
    """NaN and infinite logits, and gradients, of a padding row: its gradient is zero, the other rows'
    are what they are without it."""
    rng = np.random.default_rng([e, k])
    x = torch.from_numpy(rng.normal(0, 1.5, (40, e)).astype(np.float32)).to(dtype)
    x[1, 3], x[2, :], x[7, 0], x[8, 1] = torch.nan, torch.nan, torch.inf, -torch.inf
    x[9, :], x[39, e - 1] = torch.inf, torch.nan
    pad = [1, 2, 7, 8, 9, 39]
    valid = np.ones(40, np.uint8)
    valid[pad] = 0
    x = x.to(dev)
    r = ops.moe_route_scored(x, k, score=score, renorm=renorm, valid_rows=valid)
    g = torch.from_numpy(rng.normal(0, 1, (40, k)).astype(np.float32))
    g[pad] = torch.nan
    got = ops.moe_route_scored_backward(x, r["selected"], g.to(dev), score=score, renorm=renorm)
    assert (got[pad] == 0).all()
    rest = [i for i in range(40) if i not in pad]
    alone = ops.moe_route_scored_backward(x[rest].contiguous(), r["selected"][rest].contiguous(),
                                          g[rest].to(dev), score=score, renorm=renorm)
    assert torch.isfinite(alone).all() and torch.equal(got[rest], alone)
