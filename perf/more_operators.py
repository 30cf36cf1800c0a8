"""Layer norm, gated linear recurrence and the router's balance loss, as cases to time and compare.

What a program needs to train and serve a block of norm, recurrent mixer and routed
feed-forward, as it calls it through reimagined_amd.ops:

  norm         ops.add_layernorm: the residual add and the next block's layer norm
  norm_bwd     ops.layernorm_backward: gradients of the rows, the weight and the bias
  recur        ops.gated_recurrence: h_t = a_t h_(t-1) + u_t over a packed ragged batch,
               the decay a and the input u formed from their gates
  recur_train  the same and ops.gated_recurrence_backward, as a training step runs them
  step         ops.gated_recurrence_step: one token per sequence
  balance      ops.moe_balance_loss and ops.moe_balance_loss_backward: the loss, per-expert
               counts and mean probabilities, and the logits' gradient

With `own` false, run() computes them in plain tensor operations; with it true, it makes the
package's calls.  exact() gives the same outputs in float64.  Widths and row counts are those
of the package's configurations (d_model 1024 / 2048, inner width 2048, sequences of 64 to 2048
tokens, 60 to 256 experts) and generic ones around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_RATE = 8.0    # of the recurrence's decay
_EPS = 1e-5    # of the layer norm
_ALPHA = 0.01  # the balance loss's share of a training loss


def listed():
    return [
        # one decode step of eight users: the norm's latency counts
        dict(name="norm_decode", kind="norm", rows=8, dim=1024, dtype="bf16"),
        # the ragged prefill batch of the hybrid layer
        dict(name="norm_prefill", kind="norm", rows=40796, dim=1024, dtype="bf16"),
        # a training step at sizes that fit no vector, float32
        dict(name="norm_bwd_odd", kind="norm_bwd", rows=1021, dim=777, residual=False,
             dtype="f32"),
        # a training step's norm behind the residual's gradient
        dict(name="norm_bwd_train", kind="norm_bwd", rows=16384, dim=2048, residual=True,
             dtype="bf16"),
        # one long sequence: the work has to be split over time
        dict(name="recur_long", kind="recur", seqs=1, tokens=65536, dim=1024, initial=False,
             dtype="bf16"),
        # the ragged prefill batch of the hybrid layer, continued from kept states
        dict(name="recur_ragged", kind="recur", seqs=32, tokens=40796, dim=2048, initial=True,
             dtype="bf16"),
        # a small training batch at odd sizes, float32
        dict(name="recur_train_odd", kind="recur_train", seqs=7, tokens=1999, dim=777,
             initial=True, dtype="f32"),
        # a training step of packed sequences
        dict(name="recur_train", kind="recur_train", seqs=8, tokens=16384, dim=2048,
             initial=False, dtype="bf16"),
        # one decode step of eight users
        dict(name="step_decode", kind="step", rows=8, dim=2048, dtype="bf16"),
        # and of a large serving batch, at an odd width
        dict(name="step_batch", kind="step", rows=1000, dim=2559, dtype="f32"),
        # balance per sequence of a ragged batch with padding rows, logits left in bf16
        dict(name="balance_ragged", kind="balance", rows=4099, experts=60, k=4, score="softmax",
             seqs=17, pad=True, dtype="bf16"),
        # balance over the whole batch behind the wide sigmoid router
        dict(name="balance_wide", kind="balance", rows=16384, experts=256, k=8, score="sigmoid",
             seqs=0, pad=False, dtype="f32"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm, odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    n = _spread(rng, lo, hi)
    return n if rng.random() < 0.4 else max(lo, n // 16 * 16)


def draw(rng):
    kind = rng.choice(["norm", "norm_bwd", "norm_bwd", "recur", "recur", "recur_train",
                       "recur_train", "step", "balance", "balance"])
    dtype = rng.choice(["bf16", "f32"])
    if kind in ("norm", "norm_bwd"):
        dim = _width(rng, 32, 8192)
        c = dict(kind=kind, rows=_spread(rng, 1, min(65536, (1 << 25) // dim)), dim=dim, dtype=dtype)
        if kind == "norm_bwd":
            c["residual"] = rng.random() < 0.5
        return c
    if kind == "step":
        return dict(kind=kind, rows=_spread(rng, 1, 1000), dim=_width(rng, 64, 4096), dtype=dtype)
    if kind == "balance":
        experts = _spread(rng, 4, 256)
        rows = _spread(rng, 1, min(32768, (1 << 22) // experts))
        return dict(kind=kind, rows=rows, experts=experts, k=rng.randint(1, min(8, experts)),
                    score=rng.choice(["softmax", "sigmoid"]),
                    seqs=rng.choice([0, _spread(rng, 1, 64)]), pad=rng.random() < 0.4, dtype=dtype)
    dim = _width(rng, 64, 4096)
    tokens = _spread(rng, 1, min(65536, (1 << 25) // dim // (1 if kind == "recur" else 2)))
    return dict(kind=kind, seqs=_spread(rng, 1, 64), tokens=tokens, dim=dim,
                initial=rng.random() < 0.4, dtype=dtype)


# ---- inputs ---------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _segments(seqs, n, seed):
    """Bounds int32 [seqs + 1] of a ragged batch of n rows: cuts at random, empty sequences too."""
    rng = np.random.default_rng(seed)
    cuts = np.sort(rng.integers(0, n + 1, size=seqs - 1))
    return torch.from_numpy(np.concatenate([[0], cuts, [n]]).astype(np.int32)).cuda()


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind = case["kind"]
    dt = _DTYPES[case["dtype"]]
    st = {"case": case, "dtype": dt}
    if kind in ("norm", "norm_bwd"):
        shape = (case["rows"], case["dim"])
        # rows of a residual stream: some channels far from the others, a mean that is not zero
        stand = 1.0 + 3.0 * torch.rand((case["dim"],), generator=g, device="cuda")
        x = (_normal(g, *shape) * stand + 0.5 * _normal(g, case["dim"])).to(dt)
        st["x"] = x
        st["w"] = 1.0 + 0.2 * _normal(g, case["dim"])
        st["b"] = 0.1 * _normal(g, case["dim"])
        if kind == "norm":
            st["delta"] = _normal(g, *shape).to(dt)
        else:
            st["dy"] = (0.01 * _normal(g, *shape)).to(dt)
            st["dres"] = (0.01 * _normal(g, *shape)).to(dt) if case["residual"] else None
            f = x.float()  # the forward's statistics
            mean = f.mean(1)
            st["mean"] = mean
            st["rstd"] = torch.rsqrt((f - mean[:, None]).square().mean(1) + _EPS)
    elif kind in ("recur", "recur_train", "step"):
        shape = (case["rows"] if kind == "step" else case["tokens"], case["dim"])
        st["x"] = _normal(g, *shape).to(dt)
        st["rg"] = (1.5 * _normal(g, *shape)).to(dt)
        st["ig"] = (1.5 * _normal(g, *shape)).to(dt)
        # decays of an open gate from 0.9 to 0.999
        a = 0.9 + 0.099 * torch.rand((case["dim"],), generator=g, device="cuda")
        st["lam"] = torch.log(torch.expm1(-torch.log(a) / _RATE))
        if kind == "step":
            st["state"] = _normal(g, *shape)
            st["next"] = torch.empty_like(st["state"])
            return st
        st["cu"] = _segments(case["seqs"], case["tokens"], seed)
        st["h0"] = _normal(g, case["seqs"], case["dim"]) if case["initial"] else None
        if kind == "recur_train":
            st["dy"] = (0.01 * _normal(g, *shape)).to(dt)
    else:
        rows, experts = case["rows"], case["experts"]
        x = 1.5 * _normal(g, rows, experts) + 0.5 * _normal(g, experts)
        st["logits"] = x.to(dt)
        r = torch.arange(rows, device="cuda")
        st["valid"] = (r % 7 != 1).to(torch.uint8) if case["pad"] else None
        sel = x.sort(dim=1, descending=True).indices[:, :case["k"]].int()
        if case["pad"]:
            sel = torch.where(st["valid"].bool()[:, None], sel, -1)
        st["selected"] = sel.contiguous()
        st["cu"] = _segments(case["seqs"], rows, seed) if case["seqs"] else None
    return st


# ---- the plain forms -------------------------------------------------------------

def _plain_norm(st):
    s = (st["x"].float() + st["delta"].float()).to(st["dtype"])
    f = s.float()
    d = f - f.mean(1, keepdim=True)
    y = d * torch.rsqrt((d * d).mean(1, keepdim=True) + _EPS) * st["w"] + st["b"]
    return s, y.to(st["dtype"])


def _plain_norm_bwd(st):
    dy = st["dy"].float()
    rstd = st["rstd"][:, None]
    n = (st["x"].float() - st["mean"][:, None]) * rstd
    g = dy * st["w"]
    dx = rstd * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    if st["dres"] is not None:
        dx = dx + st["dres"].float()
    return dx.to(st["dtype"]), (dy * n).sum(0), dy.sum(0)


def _plain_gates(st):
    """a, beta, g and the two gates, float32."""
    sr = 1.0 / (1.0 + torch.exp(-st["rg"].float()))
    si = 1.0 / (1.0 + torch.exp(-st["ig"].float()))
    sp = torch.log1p(torch.exp(-st["lam"].abs())) + st["lam"].clamp_min(0.0)
    g = _RATE * sp * sr
    return torch.exp(-g), torch.sqrt(-torch.expm1(-2.0 * g)), g, sr, si


def _plain_scan(a, u):
    """h_t = a_t h_(t-1) + u_t along dim 0, by doubling the reach of every term; a and u are
    overwritten."""
    reach = 1
    while reach < a.shape[0]:
        u[reach:] = u[reach:] + a[reach:] * u[:-reach]
        a[reach:] = a[reach:] * a[:-reach]
        reach *= 2
    return u


def _bounds(st):
    """Real sequences: their numbers, first and last tokens."""
    cu = st["cu"].long()
    full = (cu[1:] > cu[:-1]).nonzero()[:, 0]
    return full, cu[full], cu[full + 1] - 1


def _plain_forward(st):
    a, beta, g, sr, si = _plain_gates(st)
    u = beta * si * st["x"].float()
    full, first, last = _bounds(st)
    carry, h = a.clone(), u.clone()
    if st["h0"] is not None:
        h[first] = h[first] + a[first] * st["h0"][full]
    carry[first] = 0.0
    h = _plain_scan(carry, h)
    final = torch.zeros((st["case"]["seqs"], a.shape[1]), device=a.device)
    if st["h0"] is not None:
        final.copy_(st["h0"])
    final[full] = h[last]
    return h, final, (a, beta, g, sr, si)


def _plain_recur(st):
    h, final, _ = _plain_forward(st)
    return h.to(st["dtype"]), final


def _plain_recur_train(st):
    h, final, (a, beta, g, sr, si) = _plain_forward(st)
    full, first, last = _bounds(st)
    before = torch.zeros_like(h)
    before[1:] = h[:-1]
    before[first] = 0.0 if st["h0"] is None else st["h0"][full]
    y = h.to(st["dtype"])
    after = torch.zeros_like(a)
    after[:-1] = a[1:]
    after[last] = 0.0
    dh = _plain_scan(after.flip(0), st["dy"].float().flip(0)).flip(0)
    x = st["x"].float()
    dx = dh * beta * si
    dig = dx * x * (1.0 - si)
    bent = torch.where(beta > 0, g * a * a / beta, 0.0)
    e = dh * (si * x * bent - a * g * before)
    drg = e * (1.0 - sr)
    sp = torch.log1p(torch.exp(-st["lam"].abs())) + st["lam"].clamp_min(0.0)
    dlam = e.sum(0) / (1.0 + torch.exp(-st["lam"])) / sp
    out = [y, final, *(t.to(st["dtype"]) for t in (dx, drg, dig)), dlam]
    if st["h0"] is not None:
        dh0 = torch.zeros_like(st["h0"])
        dh0[full] = a[first] * dh[first]
        out.append(dh0)
    return tuple(out)


def _plain_step(st):
    a, beta, _, _, si = _plain_gates(st)
    h = a * st["state"] + beta * si * st["x"].float()
    return h.to(st["dtype"]), h


def _plain_balance(st):
    c = st["case"]
    rows, experts, k = c["rows"], c["experts"], c["k"]
    x = st["logits"].float()
    if c["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
        p = s / s.sum(1, keepdim=True)
    else:
        e = torch.exp(x - x.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
    seqs = max(c["seqs"], 1)
    if st["cu"] is None:
        seq = torch.zeros(rows, dtype=torch.int64, device=x.device)
    else:
        at = torch.arange(rows, device=x.device)
        seq = (at[:, None] >= st["cu"][None, 1:]).sum(1)
    ok = (torch.ones(rows, dtype=torch.bool, device=x.device) if st["valid"] is None
          else st["valid"].bool())
    member = (seq[None, :] == torch.arange(seqs, device=x.device)[:, None]) & ok[None, :]
    tokens = member.sum(1)
    probs = member.float() @ p
    key = (seq[:, None] * experts + st["selected"].long())[ok].reshape(-1)
    counts = torch.zeros(seqs * experts, dtype=torch.int64, device=x.device)
    counts.index_add_(0, key, torch.ones_like(key))
    counts = counts.view(seqs, experts)
    n = tokens.clamp_min(1).float()[:, None]
    mean = probs / n
    some = (tokens > 0).sum().clamp_min(1).float()
    coef = experts * counts.float() / (k * n)
    loss = (coef * mean).sum() / some
    coef = (coef / (n * some))[seq]
    dx = p * (coef - (coef * p).sum(1, keepdim=True))
    if c["score"] == "sigmoid":
        dx = dx * (1.0 - s)
    dx = torch.where(ok[:, None], dx, 0.0) * _ALPHA
    return loss.reshape(1), counts.int(), tokens.int(), mean, dx.to(st["dtype"])


# ---- one pass ---------------------------------------------------------------------

def run(st):
    c = st["case"]
    kind = c["kind"]
    if not own:
        return {"norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "recur": _plain_recur,
                "recur_train": _plain_recur_train, "step": _plain_step,
                "balance": _plain_balance}[kind](st)
    from reimagined_amd import ops
    if kind == "norm":
        return ops.add_layernorm(st["x"], st["delta"], st["w"], st["b"], eps=_EPS)
    if kind == "norm_bwd":
        r = ops.layernorm_backward(st["dy"], st["x"], st["mean"], st["rstd"], st["w"],
                                   dresidual=st["dres"])
        return r["dx"], r["dweight"], r["dbias"]
    if kind == "step":
        y = ops.gated_recurrence_step(st["x"], st["rg"], st["ig"], st["lam"], st["state"],
                                      rate=_RATE, state_out=st["next"])
        return y, st["next"]
    if kind == "balance":
        f = ops.moe_balance_loss(st["logits"], st["selected"], score=c["score"],
                                 cu_seqlens=st["cu"], valid_rows=st["valid"])
        dx = ops.moe_balance_loss_backward(st["logits"], f["counts"], f["tokens"], c["k"],
                                           score=c["score"], cu_seqlens=st["cu"],
                                           valid_rows=st["valid"], dloss=_ALPHA)
        return f["loss"], f["counts"], f["tokens"], f["mean_prob"], dx
    if kind == "recur":
        return ops.gated_recurrence(st["x"], st["rg"], st["ig"], st["lam"], st["cu"], rate=_RATE,
                                    initial_state=st["h0"])
    y, final, carry = ops.gated_recurrence(st["x"], st["rg"], st["ig"], st["lam"], st["cu"],
                                           rate=_RATE, initial_state=st["h0"], want_carry=True)
    r = ops.gated_recurrence_backward(st["dy"], st["x"], st["rg"], st["ig"], st["lam"], st["cu"],
                                      carry, rate=_RATE, initial_state=st["h0"])
    out = [y, final, r["dx"], r["drg"], r["dig"], r["dlam"]]
    if st["h0"] is not None:
        out.append(r["dinitial"])
    return tuple(out)


# ---- 64 bits ----------------------------------------------------------------------

def _exact_norm(st):
    s = (st["x"].double() + st["delta"].double()).to(st["dtype"])  # what is stored is what is normed
    var, mean = torch.var_mean(s.double(), dim=1, correction=0, keepdim=True)
    y = (s.double() - mean) / torch.sqrt(var + _EPS)
    return s.double(), torch.addcmul(st["b"].double(), y, st["w"].double())


def _exact_norm_bwd(st):
    """Through the definition's Jacobian: dn, then the variance's and the mean's share."""
    x, dy = st["x"].double(), st["dy"].double()
    d = x.shape[1]
    q = st["rstd"].double()[:, None]
    far = x - st["mean"].double()[:, None]
    dn = dy * st["w"].double()
    dvar = -0.5 * (dn * far).sum(1, keepdim=True) * q ** 3
    dx = dn * q + 2.0 / d * dvar * far - (dn * q).sum(1, keepdim=True) / d
    if st["dres"] is not None:
        dx += st["dres"].double()
    return dx, torch.mv((dy * far).t().contiguous(), q[:, 0]), dy.sum(0)


def _exact_blocks(a, u):
    """h_t = a_t h_(t-1) + u_t: token after token inside blocks of about sqrt(T) tokens, all blocks
    side by side, then block after block."""
    t, d = a.shape
    size = max(1, math.isqrt(t))
    blocks = -(-t // size)
    full = blocks * size
    a = torch.cat([a, a.new_zeros(full - t, d)]).view(blocks, size, d)
    h = torch.cat([u, u.new_zeros(full - t, d)]).view(blocks, size, d)
    reach = a.clone()
    for i in range(1, size):
        h[:, i] += a[:, i] * h[:, i - 1]
        reach[:, i] *= reach[:, i - 1]
    for b in range(1, blocks):
        h[b] += reach[b] * h[b - 1, -1]
    return h.view(full, d)[:t]


def _exact_sequences(st):
    bounds = st["cu"].tolist()
    return [(s, lo, hi) for s, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])) if hi > lo]


def _exact_forward(st):
    d = {n: st[n].double() for n in ("x", "rg", "ig", "lam")}
    log_a = -_RATE * torch.nn.functional.softplus(d["lam"], threshold=700.0) * torch.sigmoid(d["rg"])
    a = log_a.exp()
    beta = (-torch.expm1(2.0 * log_a)).sqrt()
    drive = beta * torch.sigmoid(d["ig"]) * d["x"]
    keep = a.clone()
    for s, lo, hi in _exact_sequences(st):
        keep[lo] = 0.0
        if st["h0"] is not None:
            drive[lo] += a[lo] * st["h0"][s].double()
    return d, log_a, a, beta, _exact_blocks(keep, drive)


def _exact_final(st, h):
    final = (torch.zeros((st["case"]["seqs"], h.shape[1]), dtype=torch.float64, device=h.device)
             if st["h0"] is None else st["h0"].double())
    for s, lo, hi in _exact_sequences(st):
        final[s] = h[hi - 1]
    return final


def _exact_recur(st):
    h = _exact_forward(st)[-1]
    return h, _exact_final(st, h)


def _exact_recur_train(st):
    """log a = -g carries the decay's gradient: dL/dlog_a = dh (a h_before - x sigmoid(ig) a^2 /
    beta), and from there to lam and the gate through log_a = -rate softplus(lam) sigmoid(rg)."""
    d, log_a, a, beta, h = _exact_forward(st)
    t = h.shape[0]
    before = torch.cat([h.new_zeros(1, h.shape[1]), h[:-1]])
    pull = torch.cat([a[1:], a.new_zeros(1, a.shape[1])])
    for s, lo, hi in _exact_sequences(st):
        before[lo] = 0.0 if st["h0"] is None else st["h0"][s].double()
        pull[hi - 1] = 0.0
    dh = _exact_blocks(pull.flip(0), st["dy"].double().flip(0)).flip(0)
    si, sr = torch.sigmoid(d["ig"]), torch.sigmoid(d["rg"])
    dlog = dh * (a * before - torch.where(beta > 0, d["x"] * si * a * a / beta, 0.0))
    dx = dh * beta * si
    dig = dh * beta * d["x"] * si * torch.sigmoid(-d["ig"])
    drg = dlog * log_a * torch.sigmoid(-d["rg"])
    dlam = -_RATE * torch.sigmoid(d["lam"]) * (dlog * sr).sum(0)
    out = [h, _exact_final(st, h), dx, drg, dig, dlam]
    if st["h0"] is not None:
        dh0 = torch.zeros_like(st["h0"], dtype=torch.float64)
        for s, lo, hi in _exact_sequences(st):
            dh0[s] = a[lo] * dh[lo]
        out.append(dh0)
    return tuple(out)


def _exact_step(st):
    d = {n: st[n].double() for n in ("x", "rg", "ig", "lam", "state")}
    log_a = -_RATE * torch.nn.functional.softplus(d["lam"], threshold=700.0) * torch.sigmoid(d["rg"])
    h = log_a.exp() * d["state"] + (-torch.expm1(2 * log_a)).sqrt() * torch.sigmoid(d["ig"]) * d["x"]
    return h, h


def _exact_balance(st):
    """Sequence by sequence on the host; the gradient through the probabilities' Jacobian."""
    c = st["case"]
    rows, experts, k = c["rows"], c["experts"], c["k"]
    x = st["logits"].double().cpu().numpy()
    sel = st["selected"].cpu().numpy()
    ok = np.ones(rows, bool) if st["valid"] is None else st["valid"].cpu().numpy() != 0
    bounds = [0, rows] if st["cu"] is None else st["cu"].tolist()
    if c["score"] == "sigmoid":
        raw = 1.0 / (1.0 + np.exp(-x))
        slope = raw * (1.0 - raw)
    else:
        raw = np.exp(x - x.max(axis=1, keepdims=True))
        slope = raw
    total = raw.sum(axis=1, keepdims=True)
    p = raw / total
    counts = np.zeros((len(bounds) - 1, experts), np.int32)
    tokens = np.zeros(len(bounds) - 1, np.int32)
    mean = np.zeros(counts.shape)
    dx = np.zeros_like(x)
    loss, some = 0.0, 0
    for s, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
        mine = np.arange(lo, hi)[ok[lo:hi]]
        tokens[s] = len(mine)
        if not len(mine):
            continue
        some += 1
        counts[s] = np.bincount(sel[mine].reshape(-1), minlength=experts)
        mean[s] = p[mine].mean(axis=0)
        share = experts * counts[s] / (k * len(mine))
        loss += float(share @ mean[s])
        # p_e = raw_e / total: dL/draw_j = (share_j - sum_e share_e p_e) / total / N_s
        draw = (share[None, :] - (p[mine] @ share)[:, None]) / total[mine] / len(mine)
        dx[mine] = draw * slope[mine]
    loss, dx = loss / max(some, 1), dx * (_ALPHA / max(some, 1))
    return (torch.tensor([loss], dtype=torch.float64), torch.from_numpy(counts),
            torch.from_numpy(tokens), torch.from_numpy(mean), torch.from_numpy(dx))


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "norm_bwd": _exact_norm_bwd, "recur": _exact_recur,
            "recur_train": _exact_recur_train, "step": _exact_step,
            "balance": _exact_balance}[case["kind"]](st)


# ---- the work of one pass -----------------------------------------------------------

def work(case):
    kind = case["kind"]
    size = 2 if case["dtype"] == "bf16" else 4
    if kind in ("norm", "norm_bwd"):
        rows, dim = case["rows"], case["dim"]
        if kind == "norm":  # x, delta; sum, y; weight and bias
            return {"bytes": 4 * rows * dim * size + 8 * dim, "flops": 9 * rows * dim}
        return {"bytes": (4 if case["residual"] else 3) * rows * dim * size + 8 * rows + 12 * dim,
                "flops": 14 * rows * dim}
    if kind == "step":  # three inputs and the state; y and the state
        return {"bytes": case["rows"] * case["dim"] * (4 * size + 8) + 4 * case["dim"],
                "flops": 20 * case["rows"] * case["dim"]}
    if kind == "balance":  # the logits twice, their gradient, the choices
        rows, experts = case["rows"], case["experts"]
        return {"bytes": 3 * rows * experts * size + 4 * rows * case["k"]
                         + 8 * max(case["seqs"], 1) * experts, "flops": 12 * rows * experts}
    n = case["tokens"] * case["dim"]
    states = 4 * case["seqs"] * case["dim"] * (2 if case["initial"] else 1)
    if kind == "recur":  # x and two gates; y
        return {"bytes": 4 * n * size + states, "flops": 22 * n}
    return {"bytes": 11 * n * size + 2 * states, "flops": 70 * n}
