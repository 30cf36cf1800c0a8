"""Scored expert routing and 8-bit integer products, as cases to time and compare.

Six operators of a routed feed-forward with int8 experts, as a program calls them through
reimagined_amd.ops:

  route        ops.moe_route_scored: softmax or sigmoid scores, a balance bias, expert
               groups, top-k, renormalised weights, and the dispatch to expert segments
  route_bwd    ops.moe_route_scored_backward: the logits' gradient from the weights'
  combine      ops.moe_combine_topk: each row's weighted sum of its experts' rows
  combine_bwd  ops.moe_combine_topk_backward: gradients of the expert rows and the weights
  int8         ops.int8_gemm: int8 codes times int8 weights, a scale per token and channel
  experts      ops.grouped_int8_gemm: the same product for every expert's segment of rows

With `own` false, run() computes them in plain tensor operations; with it true, it makes the
package's calls.  exact() gives the same outputs in float64.  Widths and row counts are those
of the package's configurations (d_model 1024 / 2048, 4x feed-forward, 8 experts top-2, 4096
and 8192 prefill rows) and of the wider routings (60 to 256 experts) that the scored router
is for.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decode step of eight users: the router's latency counts
        dict(name="route_decode", kind="route", rows=8, experts=64, k=6, score="softmax",
             bias=False, groups=1, keep=1, best=1, renorm=True, scale=1.0, pad=False,
             dtype="f32"),
        # a ragged batch with padding rows, odd sizes, logits left in bf16, plain softmax weights
        dict(name="route_ragged", kind="route", rows=4099, experts=60, k=4, score="softmax",
             bias=True, groups=1, keep=1, best=1, renorm=False, scale=1.0, pad=True,
             dtype="bf16"),
        # prefill through a wide router: sigmoid scores, balance bias, 4 of 8 expert groups
        dict(name="route_prefill", kind="route", rows=16384, experts=256, k=8, score="sigmoid",
             bias=True, groups=8, keep=4, best=2, renorm=True, scale=2.5, pad=False,
             dtype="f32"),
        # a training step's router gradients: softmax weights as they are (every logit moves)
        dict(name="route_bwd_softmax", kind="route_bwd", rows=8192, experts=64, k=6,
             score="softmax", renorm=False, scale=1.0, pad=False, dtype="f32"),
        # and of the wide router: renormalised sigmoid weights (only the chosen logits move)
        dict(name="route_bwd_sigmoid", kind="route_bwd", rows=16384, experts=256, k=8,
             score="sigmoid", renorm=True, scale=2.5, pad=True, dtype="f32"),
        # the weighted sum behind the prefill's experts
        dict(name="combine_prefill", kind="combine", rows=8192, experts=8, k=2, dim=1024,
             pad=False, dtype="bf16"),
        # a training step's gradients through that sum, eight experts a token
        dict(name="combine_bwd", kind="combine_bwd", rows=4096, experts=64, k=8, dim=2048,
             pad=False, dtype="bf16"),
        # one token of one user through a square projection: one read of the weights
        dict(name="int8_decode", kind="int8", rows=1, k=4096, n=4096, bias=False, dtype="bf16"),
        # a short prompt at sizes that fit no tile, float32 out, with a bias
        dict(name="int8_odd", kind="int8", rows=77, k=2009, n=5125, bias=True, dtype="f32"),
        # prefill of 4096 tokens through a feed-forward sized projection
        dict(name="int8_prefill", kind="int8", rows=4096, k=4096, n=8192, bias=False,
             dtype="bf16"),
        # a decode batch of 32 users, six of 64 small experts each, up projection
        dict(name="experts_decode", kind="experts", rows=32, experts=64, top_k=6, k=1024, n=1408,
             squared_relu=True, gather=True, dtype="bf16"),
        # prefill of the routed feed-forward's up projection
        dict(name="experts_prefill", kind="experts", rows=8192, experts=8, top_k=2, k=1024,
             n=4096, squared_relu=True, gather=True, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm, odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "route", "route_bwd", "combine", "combine_bwd", "int8", "int8",
                       "int8", "experts", "experts"])
    dtype = rng.choice(["bf16", "f32"])
    if kind in ("route", "route_bwd"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _spread(rng, 8, 256 // groups) if groups > 1 else _spread(rng, 4, 256)
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(8, keep * experts // groups))
        rows = _spread(rng, 1, min(16384, 16384 * 256 // experts))
        c = dict(kind=kind, rows=rows, experts=experts, k=k,
                 score=rng.choice(["softmax", "sigmoid"]), renorm=rng.random() < 0.6,
                 scale=rng.choice([1.0, 2.5]), pad=rng.random() < 0.3, dtype=dtype)
        if kind == "route":
            c.update(bias=rng.random() < 0.6, groups=groups, keep=keep, best=rng.choice([1, 2]))
        return c
    if kind in ("combine", "combine_bwd"):
        experts = _spread(rng, 2, 256)
        k = rng.randint(1, min(8, experts))
        dim = _spread(rng, 16, 4096)
        return dict(kind=kind, rows=_spread(rng, 1, min(16384, 4096 * 8 * 2048 // (k * dim))),
                    experts=experts, k=k, dim=dim if rng.random() < 0.3 else dim // 16 * 16,
                    pad=rng.random() < 0.3, dtype=dtype)
    k = _spread(rng, 64, 8192)
    n = _spread(rng, 16, 8192)
    if rng.random() < 0.75:
        k = (k + 15) // 16 * 16
    if rng.random() < 0.75:
        n = n // 16 * 16
    if kind == "int8":
        return dict(kind=kind, rows=_spread(rng, 1, min(16384, 4096 * 4096 * 8192 // (k * n))), k=k,
                    n=n, bias=rng.random() < 0.4, dtype=dtype)
    top_k = rng.choice([1, 2, 4, 6, 8])
    experts = _spread(rng, top_k, 128)
    experts = max(top_k, min(experts, (1 << 29) // (k * n)))
    rows = _spread(rng, 1, max(1, min(8192, 8192 * 2 * 1024 * 4096 // (top_k * k * n))))
    return dict(kind=kind, rows=rows, experts=experts, top_k=top_k, k=k, n=n,
                squared_relu=rng.random() < 0.5, gather=rng.random() < 0.5, dtype=dtype)


# ---- inputs ---------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _codes(g, *shape, std):
    """int8 codes and scales of N(0, std) rows, the largest magnitude of a row at 127."""
    x = _normal(g, *shape) * std
    scale = x.abs().amax(-1) / 127.0
    return torch.round(x / scale.unsqueeze(-1)).to(torch.int8), scale


def _logits(g, case):
    """Router logits: N(0, 1.5) around expert means, some experts in favour."""
    x = 1.5 * _normal(g, case["rows"], case["experts"]) + 0.5 * _normal(g, case["experts"])
    return x.to(_DTYPES[case["dtype"]])


def _padding(case):
    """The valid-row mask: every seventh row, from the second on, is padding."""
    r = torch.arange(case["rows"], device="cuda")
    return (r % 7 != 1).to(torch.uint8) if case["pad"] else None


def _slots(g, rows, experts, k, valid):
    """A skewed routing: k different experts a row, the rows of each expert in order.
    -> selected int64 [rows, k], offsets int32, perm int32, slot_of int32 (-1 in padding rows)."""
    liked = _normal(g, rows, experts) + 0.7 * _normal(g, experts)
    selected = liked.sort(dim=1, descending=True).indices[:, :k]
    if valid is not None:
        selected = torch.where(valid.bool()[:, None], selected, -1)
    return (selected.int(), *_dispatch(selected, experts)[1:])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind = case["kind"]
    st = {"case": case, "dtype": _DTYPES[case["dtype"]]}
    if kind == "route":
        st["logits"] = _logits(g, case)
        st["bias"] = 0.1 * _normal(g, case["experts"]) if case["bias"] else None
        st["valid"] = _padding(case)
    elif kind == "route_bwd":
        st["logits"] = _logits(g, case)
        st["selected"] = _slots(g, case["rows"], case["experts"], case["k"], _padding(case))[0]
        st["dweights"] = 0.01 * _normal(g, case["rows"], case["k"])
    elif kind in ("combine", "combine_bwd"):
        _, _, st["perm"], st["slot_of"] = _slots(g, case["rows"], case["experts"], case["k"],
                                                 _padding(case))
        w = torch.rand((case["rows"], case["k"]), generator=g, device="cuda") + 0.05
        st["weights"] = w / w.sum(1, keepdim=True)
        st["expert_out"] = _normal(g, case["rows"] * case["k"], case["dim"]).to(st["dtype"])
        if kind == "combine_bwd":
            st["dout"] = (0.01 * _normal(g, case["rows"], case["dim"])).to(st["dtype"])
    elif kind == "int8":
        st["q"], st["act_scale"] = _codes(g, case["rows"], case["k"], std=1.0)
        st["w"], st["w_scale"] = _codes(g, case["n"], case["k"], std=0.02)
        st["bias"] = 0.1 * _normal(g, case["n"]) if case["bias"] else None
    else:
        _, st["offsets"], st["perm"], _ = _slots(g, case["rows"], case["experts"], case["top_k"],
                                                 None)
        slots = case["rows"] * case["top_k"]
        st["q"], st["act_scale"] = _codes(g, case["rows"] if case["gather"] else slots, case["k"],
                                          std=1.0)
        st["w"], st["w_scale"] = _codes(g, case["experts"], case["n"], case["k"], std=0.02)
        if not case["gather"]:
            st["perm"] = None
    return st


# ---- the plain forms -------------------------------------------------------------

def _dispatch(selected, experts):
    """Expert-major, rows-ascending slots of int64 selections [rows, k] (-1: none)
    -> counts, offsets, perm (-1 past the last slot), slot_of, int32."""
    rows, k = selected.shape
    key = torch.where(selected < 0, experts, selected).reshape(-1)
    order = key.sort(stable=True).indices
    counts = (key[:, None] == torch.arange(experts, device=key.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    at = torch.arange(rows * k, device=key.device)
    perm = torch.where(at < offsets[-1], order // k, -1)
    slot_of = torch.empty_like(at)
    slot_of[order] = at
    slot_of = torch.where(selected < 0, -1, slot_of.view(rows, k))
    return counts.int(), offsets.int(), perm.int(), slot_of.int()


def _scores(x, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _plain_route(st):
    c = st["case"]
    rows, experts, k, groups = c["rows"], c["experts"], c["k"], c["groups"]
    # 64 bits: scores that lie next to each other decide which expert is chosen
    x = st["logits"].double()
    s = _scores(x, c["score"])
    choice = s if st["bias"] is None else s + st["bias"].double()
    if groups > 1:
        per = choice.view(rows, groups, experts // groups).sort(dim=2, descending=True).values
        kept = per[:, :, :c["best"]].sum(2).sort(dim=1, descending=True, stable=True).indices
        open_ = torch.zeros((rows, groups), dtype=torch.bool, device=x.device)
        open_.scatter_(1, kept[:, :c["keep"]], True)
        choice = torch.where(open_.repeat_interleave(experts // groups, dim=1), choice, -math.inf)
    selected = choice.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, selected)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = w * c["scale"]
    if st["valid"] is not None:
        ok = st["valid"].bool()[:, None]
        selected = torch.where(ok, selected, -1)
        w = torch.where(ok, w, 0.0)
    return (w.float(), selected.int(), *_dispatch(selected, experts))


def _plain_route_bwd(st):
    c = st["case"]
    x = st["logits"].float()
    sel = st["selected"].long()
    dw = torch.where(sel < 0, 0.0, st["dweights"]) * c["scale"]
    at = sel.clamp_min(0)
    s = _scores(x, c["score"])
    chosen = s.gather(1, at)
    if c["renorm"]:
        total = chosen.sum(1, keepdim=True)
        ds = (dw - (dw * chosen).sum(1, keepdim=True) / total) / total
    else:
        ds = dw
    dscore = torch.zeros_like(x).scatter_(1, at, torch.where(sel < 0, 0.0, ds))
    if c["score"] == "sigmoid":
        dx = dscore * s * (1.0 - s)
    else:
        dx = s * (dscore - (dscore * s).sum(1, keepdim=True))
    return dx.to(st["dtype"])


def _plain_combine(st):
    c = st["case"]
    slot = st["slot_of"].long()
    rows = st["expert_out"].float()[slot.clamp_min(0).reshape(-1)].view(c["rows"], c["k"], c["dim"])
    w = torch.where(slot < 0, 0.0, st["weights"])
    return (rows * w[:, :, None]).sum(1).to(st["dtype"])


def _plain_combine_bwd(st):
    c = st["case"]
    slot = st["slot_of"].long()
    at = slot.clamp_min(0).reshape(-1)
    dout = st["dout"].float()[:, None, :]
    rows = st["expert_out"].float()[at].view(c["rows"], c["k"], c["dim"])
    dw = torch.where(slot < 0, 0.0, (rows * dout).sum(2))
    drows = (st["weights"][:, :, None] * dout).reshape(-1, c["dim"]).to(st["dtype"])
    dexpert = torch.zeros_like(st["expert_out"])
    real = (slot >= 0).reshape(-1)
    dexpert[at[real]] = drows[real]
    return dexpert, dw


def _plain_product(q, act_scale, w, w_scale, bias, squared_relu):
    y = (q.float() @ w.float().t()) * act_scale[:, None] * w_scale[None, :]
    if bias is not None:
        y = y + bias
    if squared_relu:
        y = y.clamp_min(0.0)
        y = y * y
    return y


def _plain_int8(st):
    return _plain_product(st["q"], st["act_scale"], st["w"], st["w_scale"], st["bias"],
                          False).to(st["dtype"])


def _plain_experts(st):
    c = st["case"]
    out = torch.empty((c["rows"] * c["top_k"], c["n"]), dtype=st["dtype"], device="cuda")
    bounds = st["offsets"].tolist()
    for e in range(c["experts"]):
        lo, hi = bounds[e], bounds[e + 1]
        if lo < hi:
            rows = slice(lo, hi) if st["perm"] is None else st["perm"][lo:hi].long()
            out[lo:hi] = _plain_product(st["q"][rows], st["act_scale"][rows], st["w"][e],
                                        st["w_scale"][e], None, c["squared_relu"])
    return out


# ---- one pass ---------------------------------------------------------------------

def run(st):
    c = st["case"]
    kind = c["kind"]
    if not own:
        return {"route": _plain_route, "route_bwd": _plain_route_bwd, "combine": _plain_combine,
                "combine_bwd": _plain_combine_bwd, "int8": _plain_int8,
                "experts": _plain_experts}[kind](st)
    from reimagined_amd import ops
    if kind == "route":
        r = ops.moe_route_scored(st["logits"], c["k"], score=c["score"], bias=st["bias"],
                                 groups=c["groups"], group_keep=c["keep"], group_best=c["best"],
                                 renorm=c["renorm"], scale=c["scale"], valid_rows=st["valid"])
        return tuple(r[n] for n in ("weights", "selected", "counts", "offsets", "perm", "slot_of"))
    if kind == "route_bwd":
        return ops.moe_route_scored_backward(st["logits"], st["selected"], st["dweights"],
                                             score=c["score"], renorm=c["renorm"],
                                             scale=c["scale"])
    if kind == "combine":
        return ops.moe_combine_topk(st["expert_out"], st["slot_of"], st["weights"],
                                    out_dtype=st["dtype"])
    if kind == "combine_bwd":
        return ops.moe_combine_topk_backward(st["dout"], st["expert_out"], st["slot_of"],
                                             st["weights"], perm=st["perm"])
    if kind == "int8":
        return ops.int8_gemm(st["q"], st["act_scale"], st["w"], st["w_scale"], bias=st["bias"],
                             out_dtype=st["dtype"])
    return ops.grouped_int8_gemm(st["q"], st["act_scale"], st["w"], st["w_scale"], st["offsets"],
                                 perm=st["perm"], squared_relu=c["squared_relu"],
                                 out_dtype=st["dtype"])


# ---- 64 bits ----------------------------------------------------------------------

def _host(t):
    return None if t is None else (t.double() if t.is_floating_point() else t).cpu().numpy()


def _exact_scores(x, score):
    with np.errstate(over="ignore"):
        if score == "sigmoid":
            return 1.0 / (1.0 + np.exp(-x))
        e = np.exp(x - x.max(axis=1, keepdims=True))
        return e / e.sum(axis=1, keepdims=True)


def _exact_route(st):
    """Selection by lexicographic sorts (value descending, index ascending); the slots from a
    running count per expert over the rows in order."""
    c = st["case"]
    rows, experts, k, groups = c["rows"], c["experts"], c["k"], c["groups"]
    s = _exact_scores(_host(st["logits"]), c["score"])
    choice = s if st["bias"] is None else s + _host(st["bias"])[None, :]
    if groups > 1:
        per = choice.reshape(rows, groups, -1)
        top = -np.sort(-per, axis=2)[:, :, :c["best"]].sum(axis=2)
        rank = np.argsort(np.argsort(-top, axis=1, kind="stable"), axis=1)
        choice = np.where((rank < c["keep"])[:, :, None], per, -np.inf).reshape(rows, experts)
    sel = np.argsort(-choice, axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(s, sel, axis=1)
    if c["renorm"]:
        w = w / w.sum(axis=1, keepdims=True)
    w = w * c["scale"]
    ok = np.ones(rows, bool) if st["valid"] is None else _host(st["valid"]) != 0
    w[~ok] = 0.0
    hits = np.zeros((rows, experts), np.int64)
    np.put_along_axis(hits, sel, 1, axis=1)
    hits[~ok] = 0
    counts = hits.sum(axis=0)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    slot = np.take_along_axis(offsets[:-1] + np.cumsum(hits, axis=0) - 1, sel, axis=1)
    slot = np.where(ok[:, None], slot, -1)
    perm = np.full(rows * k, -1, np.int64)
    perm[slot[ok].reshape(-1)] = np.repeat(np.arange(rows)[ok], k)
    sel = np.where(ok[:, None], sel, -1)
    ints = [torch.from_numpy(a.astype(np.int32)) for a in (sel, counts, offsets, perm, slot)]
    return (torch.from_numpy(w), *ints)


def _exact_route_bwd(st):
    """Through the Jacobians of the weights by the logits: with p the scores and W the sum over
    the chosen, dw_i / ds_j = (1[i = j] - w_i) / W where renormalised; ds/dx = s (1 - s), or
    p_i (1[i = j] - p_j) for the softmax."""
    c = st["case"]
    x, sel, dw = _host(st["logits"]), _host(st["selected"]), _host(st["dweights"])
    none = sel < 0
    at = np.where(none, 0, sel)
    dw = np.where(none, 0.0, dw) * c["scale"]
    s = _exact_scores(x, c["score"])
    t = np.where(none, 0.0, np.take_along_axis(s, at, axis=1))
    total = np.where(none.all(axis=1), 1.0, t.sum(axis=1))[:, None]
    g = np.zeros_like(x)
    if c["renorm"]:
        w = t / total
        # sum_i dw_i w_i (1[i = j] - w_j), divided by the score where its own factor enters
        grad_log = w * (dw - (dw * w).sum(axis=1, keepdims=True))
        if c["score"] == "sigmoid":
            grad_log = grad_log * (1.0 - np.take_along_axis(s, at, axis=1))
        np.add.at(g, (np.arange(len(x))[:, None], at), np.where(none, 0.0, grad_log))
    elif c["score"] == "sigmoid":
        np.add.at(g, (np.arange(len(x))[:, None], at), dw * t * (1.0 - t))
    else:
        np.add.at(g, (np.arange(len(x))[:, None], at), dw * t)
        g -= s * (dw * t).sum(axis=1, keepdims=True)
    return torch.from_numpy(g)


def _exact_combine(st):
    c = st["case"]
    out = torch.zeros((c["rows"], c["dim"]), dtype=torch.float64, device="cuda")
    for i in range(c["k"]):
        r = (st["slot_of"][:, i] >= 0).nonzero()[:, 0]
        rows = st["expert_out"][st["slot_of"][r, i].long()].double()
        out[r] += rows * st["weights"][r, i].double()[:, None]
    return out


def _exact_combine_bwd(st):
    c = st["case"]
    dexpert = torch.zeros(st["expert_out"].shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros((c["rows"], c["k"]), dtype=torch.float64, device="cuda")
    for i in range(c["k"]):
        r = (st["slot_of"][:, i] >= 0).nonzero()[:, 0]
        slot = st["slot_of"][r, i].long()
        d = st["dout"][r].double()
        dexpert[slot] = d * st["weights"][r, i].double()[:, None]
        dw[r, i] = (d * st["expert_out"][slot].double()).sum(1)
    return dexpert, dw


def _exact_product(q, act_scale, w, w_scale, bias, squared_relu):
    scaled = torch.mm(q.double() * act_scale.double()[:, None],
                      (w.double() * w_scale.double()[:, None]).t().contiguous())
    if bias is not None:
        scaled = scaled + bias.double()[None, :]
    return torch.square(torch.relu(scaled)) if squared_relu else scaled


def _exact_int8(st):
    return _exact_product(st["q"], st["act_scale"], st["w"], st["w_scale"], st["bias"], False)


def _exact_experts(st):
    c = st["case"]
    slots = c["rows"] * c["top_k"]
    at = torch.arange(slots, device="cuda") if st["perm"] is None else st["perm"].long()
    out = torch.empty((slots, c["n"]), dtype=torch.float64, device="cuda")
    expert = torch.bucketize(torch.arange(slots, device="cuda"), st["offsets"][1:].long(),
                             right=True)
    for e in torch.unique(expert).tolist():
        mine = (expert == e).nonzero()[:, 0]
        out[mine] = _exact_product(st["q"][at[mine]], st["act_scale"][at[mine]], st["w"][e],
                                   st["w_scale"][e], None, c["squared_relu"])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"route": _exact_route, "route_bwd": _exact_route_bwd, "combine": _exact_combine,
            "combine_bwd": _exact_combine_bwd, "int8": _exact_int8,
            "experts": _exact_experts}[case["kind"]](st)


# ---- the work of one pass -----------------------------------------------------------

def work(case):
    kind, rows = case["kind"], case["rows"]
    size = 2 if case["dtype"] == "bf16" else 4
    if kind in ("route", "route_bwd"):
        e, k = case["experts"], case["k"]
        if kind == "route":  # logits; weights, selections, slots and the permutation; the segments
            return {"bytes": rows * e * size + rows * k * 16 + 8 * e, "flops": 4 * rows * e}
        chosen_only = case["renorm"] or case["score"] == "sigmoid"
        read = rows * (min(k, e) if chosen_only else e) * size
        return {"bytes": read + rows * k * 8 + rows * e * size,
                "flops": 4 * rows * (k if chosen_only else e)}
    if kind == "combine":
        k, dim = case["k"], case["dim"]
        return {"bytes": rows * dim * size * (k + 1) + rows * k * 8, "flops": 2 * rows * k * dim}
    if kind == "combine_bwd":
        k, dim = case["k"], case["dim"]
        return {"bytes": rows * dim * size * (2 * k + 1) + rows * k * 12,
                "flops": 3 * rows * k * dim}
    k, n = case["k"], case["n"]
    if kind == "int8":
        return {"bytes": rows * k + n * k + rows * n * size + 4 * (rows + 2 * n),
                "flops": 2 * rows * k * n}
    slots = rows * case["top_k"]
    return {"bytes": (rows if case["gather"] else slots) * (k + 4)
                     + min(case["experts"], slots) * n * (k + 4) + slots * (n * size + 4),
            "flops": 2 * slots * k * n}
