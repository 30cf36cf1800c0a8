"""The operators of scored routing and int8 experts together, as the layers run them: the whole
feed-forward against the oracle's quantizer and the definitions (codes and expert rows bit for
bit, the combine to its rounding), its router's gradients, the hybrid block on top of it, other
streams, and captured graphs replayed between eager work."""
import numpy as np
import pytest
import torch

from reimagined_amd import layers, ops, workloads
from reimagined_amd.layers import HybridBlock, Int8Linear, Int8MoEFFN

from test_gpu_int8_gemm import product
from test_gpu_route_scored import dispatch_ref, grad64, route64, rtol

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def t(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def codes(orc, x, rms):
    return orc.quantize_act(orc.rmsnorm(x) if rms else x, 8)


def experts(rng, e, ff, d):
    return (rng.normal(0, 0.05, (e, ff, d)).astype(np.float32),
            rng.normal(0, 0.05, (e, d, ff)).astype(np.float32))


@pytest.mark.parametrize("m,k,n", [(1, 64, 48), (7, 192, 33), (150, 256, 130)])
@pytest.mark.parametrize("rms", [False, True])
def test_int8_linear(dev, orc, m, k, n, rms):
    rng = np.random.default_rng([m, k, n])
    w, x, b = (rng.normal(0, 1, s).astype(np.float32) for s in ((n, k), (m, k), (n,)))
    lin = Int8Linear(w, dev, bias=b, rms_input=rms)
    wq, ws = orc.quantize_act(w, 8)
    assert np.array_equal(lin.w.cpu().numpy(), wq) and np.array_equal(lin.w_scale.cpu().numpy(), ws)
    q, s = codes(orc, x, rms)
    got = lin.forward(t(x, dev))
    np.testing.assert_array_equal(got.cpu().numpy(), product(q, s, wq, ws, b))
    # against float: half a step (1 / 254 of a row's largest) of either operand at each of K terms
    xr = orc.rmsnorm(x) if rms else x
    err = np.abs(got.cpu().numpy() - (xr.astype(np.float64) @ w.T.astype(np.float64) + b))
    step = (np.abs(xr).max(1)[:, None] * np.abs(w).sum(1)[None] + np.abs(w).max(1)[None] * np.abs(xr).sum(1)[:, None])
    assert (err <= 1.05 * step / 254 + 1e-4).all()


@pytest.mark.parametrize("rows,e,d,ff,k,routing", [
    (1, 8, 128, 256, 2, {}),
    (37, 6, 64, 96, 3, dict(score="sigmoid", scale=2.5)),
    (300, 16, 128, 192, 4, dict(score="sigmoid", groups=4, group_keep=2, bias=True)),
    (700, 70, 64, 80, 2, dict(renorm=False)),
])
@pytest.mark.parametrize("pad", [False, True])
@pytest.mark.parametrize("rms", [False, True])
def test_feed_forward(dev, orc, rows, e, d, ff, k, routing, pad, rms):
    rng = np.random.default_rng([rows, e, d])
    routing = dict(routing)
    bias = rng.normal(0, 0.1, e).astype(np.float32) if routing.pop("bias", False) else None
    up, down = experts(rng, e, ff, d)
    x = rng.normal(0, 1, (rows, d)).astype(np.float32)
    logits = rng.normal(0, 1.5, (rows, e)).astype(np.float32)
    valid = (rng.random(rows) < 0.8).astype(np.uint8) if pad else None
    moe = Int8MoEFFN(up, down, dev, k=k, balance_bias=bias, rms_input=rms, **routing)
    res = moe.forward(t(x, dev), t(logits, dev), valid_rows=valid)
    want_w, want_sel = route64(logits.astype(np.float64), k, routing.get("score", "softmax"), bias,
                               routing.get("groups", 1), routing.get("group_keep", 1), 2,
                               routing.get("renorm", True), routing.get("scale", 1.0), valid)
    counts, offsets, perm, slot_of = dispatch_ref(want_sel, e)
    np.testing.assert_array_equal(res["selected"].cpu().numpy(), want_sel)
    np.testing.assert_array_equal(res["perm"].cpu().numpy(), perm)
    np.testing.assert_array_equal(res["slot_of"].cpu().numpy(), slot_of)
    np.testing.assert_allclose(res["weights"].cpu().numpy(), want_w, rtol=rtol(logits), atol=1e-37)
    total = offsets[-1]
    uq, us = orc.quantize_act(up.reshape(-1, d), 8)
    dq, ds = orc.quantize_act(down.reshape(-1, ff), 8)
    uq, us, dq, ds = uq.reshape(e, ff, d), us.reshape(e, ff), dq.reshape(e, d, ff), ds.reshape(e, d)
    q, s = codes(orc, x, rms)
    h = np.zeros((total, ff), np.float32)
    o = np.zeros((total, d), np.float32)
    for i in range(e):
        seg = slice(offsets[i], offsets[i + 1])
        if offsets[i] < offsets[i + 1]:
            h[seg] = product(q[perm[seg]], s[perm[seg]], uq[i], us[i], None, True)
            hq, hs = codes(orc, h[seg], rms)
            o[seg] = product(hq, hs, dq[i], ds[i])
    np.testing.assert_array_equal(res["h"].cpu().numpy()[:total], h)
    np.testing.assert_array_equal(res["o"].cpu().numpy()[:total], o)
    w = res["weights"].double().cpu().numpy() * (slot_of >= 0)
    rows_o = o.astype(np.float64)[np.maximum(slot_of, 0)] if total else np.zeros((rows, k, d))
    out = (rows_o * w[:, :, None]).sum(1)
    mag = (np.abs(rows_o) * w[:, :, None]).sum(1)
    assert (np.abs(res["out"].double().cpu().numpy() - out) <= (k + 1) * 2.0**-24 * mag).all()
    # the router's gradients, through the combine and the weights
    dout = rng.normal(0, 1, (rows, d)).astype(np.float32)
    g = moe.router_backward(t(logits, dev), res, t(dout, dev))
    dw = (rows_o * dout.astype(np.float64)[:, None, :]).sum(2) * (slot_of >= 0)
    mag = (np.abs(rows_o) * np.abs(dout)[:, None, :]).sum(2)
    assert (np.abs(g["dweights"].cpu().numpy() - dw) <= (d / 64 + 17) * 2.0**-24 * mag).all()
    want = grad64(logits.astype(np.float64), want_sel, g["dweights"].double().cpu().numpy(),
                  routing.get("score", "softmax"), routing.get("renorm", True), routing.get("scale", 1.0))
    lim = 2 * (rtol(logits) + 24 * 2.0**-24) * routing.get("scale", 1.0) * \
        np.abs(g["dweights"].cpu().numpy()).max(1, keepdims=True)
    assert (np.abs(g["dlogits"].cpu().numpy() - want) <= lim).all()
    do = g["do"].cpu().numpy()
    assert (do[total:] == 0).all()
    for r in range(rows):
        for i in range(k):
            if slot_of[r, i] >= 0:
                np.testing.assert_allclose(do[slot_of[r, i]], w[r, i] * dout[r], rtol=2.0**-23)


def test_all_rows_padding(dev):
    rng = np.random.default_rng(1)
    up, down = experts(rng, 4, 96, 64)
    moe = Int8MoEFFN(up, down, dev)
    x, logits = torch.randn(9, 64, device=dev), torch.randn(9, 4, device=dev)
    res = moe.forward(x, logits, valid_rows=np.zeros(9, np.uint8))
    assert (res["out"] == 0).all() and res["offsets"].tolist() == [0] * 5
    g = moe.router_backward(logits, res, torch.randn(9, 64, device=dev))
    assert (g["dlogits"] == 0).all() and (g["dweights"] == 0).all() and (g["do"] == 0).all()


def test_hybrid_block(dev):
    """HybridBlock(moe=Int8MoEFFN): the block around the feed-forward is the one it was."""
    rng = np.random.default_rng(5)
    params, inp = workloads.config4(seed=13, num_seqs=3, d_model=128, lo=5, hi=60)
    up, down = experts(rng, 6, 256, 128)
    gate_w = (rng.standard_normal((6, 128)) / 11).astype(np.float32)
    moe = Int8MoEFFN(list(up), list(down), dev, k=2, score="sigmoid")
    blk = HybridBlock(params, None, None, dev, gate_w=gate_w, moe=moe)
    tb = lambda a: t(a, dev).to(BF16)
    res = blk.forward(tb(inp["x"]), tb(inp["dt"]), tb(inp["B"]), tb(inp["C"]), t(inp["cu_seqlens"], dev))
    ff = moe.forward(res["f"], res["logits"], out_dtype=BF16)["out"]
    assert torch.equal(ff, res["ff"])
    assert torch.equal(res["out"], (res["residual"].float() + ff.float()).to(BF16))


def test_refusals(dev):
    rng = np.random.default_rng(2)
    up, down = experts(rng, 4, 96, 64)
    with pytest.raises(ValueError, match="agree"):
        Int8MoEFFN(up, down[:, :, :80], dev)
    with pytest.raises(ValueError, match="outputs"):
        layers.quantize_weights_i8(np.zeros(5, np.float32), dev)
    moe = Int8MoEFFN(up, down, dev, k=5)
    with pytest.raises(ValueError, match="experts"):
        moe.forward(torch.zeros(3, 64, device=dev), torch.zeros(3, 4, device=dev))
    with pytest.raises(ValueError, match="logits"):
        moe.forward(torch.zeros(3, 64, device=dev), torch.zeros(3, 5, device=dev))
    q, s = torch.zeros(4, 8, dtype=torch.int8, device=dev), torch.zeros(4, device=dev)
    w, ws = torch.zeros(3, 8, dtype=torch.int8, device=dev), torch.zeros(3, device=dev)
    for bad, text in ((dict(q=q[:, ::2], w=w[:, ::2]), "contiguous"), (dict(act_scale=s[:3]), "act_scale"),
                      (dict(w_scale=ws.double()), "w_scale"), (dict(bias=torch.zeros(4, device=dev)), "bias"),
                      (dict(act_scale=s.cpu()), "device"), (dict(out_dtype=torch.float16), "out_dtype"),
                      (dict(q=q.float()), "q must be")):
        with pytest.raises(ValueError, match=text):
            ops.int8_gemm(**{**dict(q=q, act_scale=s, w=w, w_scale=ws), **bad})
    x = torch.zeros(4, 8, device=dev)
    for bad, text in ((dict(score="tanh"), "score"), (dict(bias=torch.zeros(7, device=dev)), "bias"),
                      (dict(valid_rows=np.array([1, 2, 0, 1])), "mask"), (dict(groups=3), "groups"),
                      (dict(k=0), "0 < k"), (dict(groups=4, group_keep=1, k=3), "kept groups")):
        with pytest.raises(ValueError, match=text):
            ops.moe_route_scored(**{**dict(logits=x, k=2), **bad})
    with pytest.raises(ValueError, match="column stride"):
        ops.moe_route_scored(torch.zeros(8, 4, device=dev).t(), 2)
    sel = torch.zeros(4, 2, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="dweights"):
        ops.moe_route_scored_backward(x, sel, torch.zeros(4, 3, device=dev))
    y = torch.zeros(8, 16, device=dev)
    with pytest.raises(ValueError, match="weights"):
        ops.moe_combine_topk(y, sel, torch.zeros(4, 3, device=dev))
    with pytest.raises(ValueError, match="dout"):
        ops.moe_combine_topk_backward(torch.zeros(3, 16, device=dev), y, sel, torch.zeros(4, 2, device=dev))


def test_on_a_side_stream(dev):
    """Work on a stream that is current but not the default one, ordered by the caller."""
    rng = np.random.default_rng(3)
    up, down = experts(rng, 8, 256, 128)
    moe = Int8MoEFFN(up, down, dev, k=2)
    x, logits = torch.randn(400, 128, device=dev), torch.randn(400, 8, device=dev)
    want = moe.forward(x, logits)["out"].clone()
    s = torch.cuda.Stream()
    for _ in range(3):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            big = torch.randn(2048, 2048, device=dev)
            for _ in range(4):
                big = big @ big * 1e-3
            late = x + 0 * big[0, 0].nan_to_num(0.0, 0.0, 0.0)
            got = moe.forward(late, logits)["out"]
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [3, 90, 1500])
def test_graph_replay(dev, rows):
    """Forward and router gradients captured once; replayed on new inputs between eager calls of
    other sizes, two graphs of one layer in turn."""
    rng = np.random.default_rng(rows)
    up, down = experts(rng, 12, 192, 128)
    moe = Int8MoEFFN(up, down, dev, k=3, score="sigmoid", groups=4, group_keep=2,
                     balance_bias=rng.normal(0, 0.1, 12))

    def work(x, logits, dout):
        res = moe.forward(x, logits)
        g = moe.router_backward(logits, res, dout)
        return res["out"], res["perm"], g["dlogits"], g["do"]

    def inputs(seed, n):
        g = torch.Generator(dev).manual_seed(seed)
        return [torch.randn(n, c, device=dev, generator=g) for c in (128, 12, 128)]

    graphs = []
    for i in range(2):
        static = inputs(i, rows)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(*static)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work(*static)
        graphs.append((g, static, out))
    for rep in range(4):
        for i, (g, static, out) in enumerate(graphs):
            fresh = inputs(10 + 2 * rep + i, rows)
            want = [v.clone() for v in work(*fresh)]
            for a, b in zip(static, fresh):
                a.copy_(b)
            work(*inputs(99, rows + 7))
            for v in out:
                v.fill_(3)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), f"replay {rep} of graph {i}"


def test_same_bits_every_time(dev):
    rng = np.random.default_rng(4)
    up, down = experts(rng, 16, 256, 128)
    moe = Int8MoEFFN(up, down, dev, k=4)
    x, logits, dout = (torch.randn(2000, c, device=dev) for c in (128, 16, 128))
    first = None
    for _ in range(5):
        res = moe.forward(x, logits)
        g = moe.router_backward(logits, res, dout)
        now = [res["out"], res["weights"], res["slot_of"], g["dlogits"], g["dweights"], g["do"]]
        if first is None:
            first = [v.clone() for v in now]
        assert all(torch.equal(a, b) for a, b in zip(now, first))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_router_gradient_of_padding_rows(dev, score, renorm):
    """Padding rows whose logits and output gradients are NaN or infinite leave the gate's gradient,
    dlogits^T x, what it is without them."""
    rng = np.random.default_rng(8)
    up, down = experts(rng, 6, 96, 64)
    moe = Int8MoEFFN(up, down, dev, k=2, score=score, renorm=renorm)
    x, logits, dout = (torch.randn(20, c, device=dev) for c in (64, 6, 64))
    pad, rest = [0, 5, 19], [i for i in range(20) if i not in (0, 5, 19)]
    logits[0, 2], logits[5], logits[19, 0] = torch.nan, torch.inf, -torch.inf
    logits[19, 1] = torch.inf
    dout[pad] = torch.nan
    valid = np.ones(20, np.uint8)
    valid[pad] = 0
    g = moe.router_backward(logits, moe.forward(x, logits, valid_rows=valid), dout)
    part = [v[rest].contiguous() for v in (x, logits, dout)]
    want = moe.router_backward(part[1], moe.forward(part[0], part[1]), part[2])
    assert (g["dlogits"][pad] == 0).all() and (g["dweights"][pad] == 0).all()
    assert torch.isfinite(want["dlogits"]).all() and torch.equal(g["dlogits"][rest], want["dlogits"])
