"""Layer norm and its gradients against float64: every row shape the kernels choose between, odd
lengths and alignments, types, absent weights, captured calls."""
import numpy as np
import pytest
import torch

import train_ref as ref
from reimagined_amd import ops
from reimagined_amd._lib import call

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
# one length, tails of each vector, every number of threads and pieces a row takes, past the registers
SIZES = [(1, 1), (3, 7), (5, 8), (70, 64), (33, 65), (9, 129), (130, 250), (6, 264), (4, 512), (11, 777),
         (300, 1024), (7, 1535), (5, 2048), (3, 2049), (2, 4100), (2, 6150), (3, 8192), (2, 8200),
         (2, 16384), (2, 16391), (1, 33000)]


def rows(rng, n, dim, dtype, dev, scale=1.0):
    x = rng.normal(0.3, 1.0, (n, dim)) * rng.uniform(0.5, 3.0, dim) * scale
    t = torch.from_numpy(x.astype(np.float32)).to(DT[dtype])
    return t.to(dev), t.double().numpy()


def vec(rng, dim, dev, mean):
    v = rng.normal(mean, 0.3, dim).astype(np.float32)
    return torch.from_numpy(v).to(dev), v.astype(np.float64)


def near(got, want, lim, dtype="f32", what=""):
    got = got.double().cpu().numpy()
    bound = lim + ref.HALF_STEP[dtype] * np.abs(want) * (1 + 2.0**-7) + 1e-37
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / bound)))


@pytest.mark.parametrize("n,dim", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("parts", ["wb", "w", "b", ""])
def test_forward(dev, n, dim, dtype, parts):
    rng = np.random.default_rng([n, dim])
    x, x64 = rows(rng, n, dim, dtype, dev)
    w, w64 = vec(rng, dim, dev, 1.0) if "w" in parts else (None, None)
    b, b64 = vec(rng, dim, dev, 0.0) if "b" in parts else (None, None)
    other = "bf16" if dtype == "f32" else "f32"
    want, mean, rstd, lim, dmean, drel = ref.layernorm(x64, w64, b64, 1e-5)
    for odt in (dtype, other):
        y, m, q = ops.layernorm(x, w, b, out_dtype=DT[odt], want_stats=True)
        assert y.dtype == DT[odt]
        near(y, want, lim, odt, "y")
        near(m, mean, dmean, what="mean")
        near(q, rstd, drel * rstd, what="rstd")


@pytest.mark.parametrize("n,dim", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_add(dev, n, dim, dtype):
    rng = np.random.default_rng([n, dim, 1])
    x, _ = rows(rng, n, dim, dtype, dev)
    d, _ = rows(rng, n, dim, dtype, dev)
    w, w64 = vec(rng, dim, dev, 1.0)
    b, b64 = vec(rng, dim, dev, 0.0)
    res, y = ops.add_layernorm(x, d, w, b)
    assert torch.equal(res, x + d)
    want, *_, = ref.layernorm(res.double().cpu().numpy(), w64, b64, 1e-5)
    near(y, want, ref.layernorm(res.double().cpu().numpy(), w64, b64, 1e-5)[3], dtype)


@pytest.mark.parametrize("n,dim", SIZES + [(3000, 100), (1025, 512), (2100, 2048)])
@pytest.mark.parametrize("dtype,gdtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("residual", [False, True])
def test_backward(dev, n, dim, dtype, gdtype, residual):
    rng = np.random.default_rng([n, dim, 2])
    x, x64 = rows(rng, n, dim, dtype, dev)
    dy, dy64 = rows(rng, n, dim, gdtype, dev, 0.01)
    w, w64 = vec(rng, dim, dev, 1.0) if not (residual and dim % 2) else (None, None)
    dres, dres64 = rows(rng, n, dim, dtype, dev, 0.01) if residual else (None, None)
    _, mean, rstd = ops.layernorm(x, w, want_stats=True)
    r = ops.layernorm_backward(dy, x, mean, rstd, w, dresidual=dres)
    dx, lim, dw, dwlim, db, dblim = ref.layernorm_backward(
        dy64, x64, mean.double().cpu().numpy(), rstd.double().cpu().numpy(), w64, dres64)
    near(r["dx"], dx, lim, dtype, "dx")
    near(r["dweight"], dw, dwlim, what="dweight")
    near(r["dbias"], db, dblim, what="dbias")
    again = ops.layernorm_backward(dy, x, mean, rstd, w, dresidual=dres)
    assert all(torch.equal(r[k], again[k]) for k in r)
    assert torch.equal(ops.layernorm_backward(dy, x, mean, rstd, w, dresidual=dres,
                                              want_params=False)["dx"], r["dx"])


@pytest.mark.parametrize("dim", [8, 100, 512, 1000, 2048, 5000, 17000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_any_alignment(dev, dim, dtype):
    """Rows that start one element past an aligned address, the sum written over delta."""
    rng = np.random.default_rng([dim, 3])
    n = 5
    x, _ = rows(rng, n, dim, dtype, dev)
    d, _ = rows(rng, n, dim, dtype, dev)
    w, _ = vec(rng, dim, dev, 1.0)
    res, y, mean, rstd = ops.add_layernorm(x, d, w, want_stats=True)

    def off(t):
        b = torch.full((n * dim + 9,), 7.0, dtype=t.dtype, device=dev)
        v = b[1:1 + n * dim].view(n, dim)
        v.copy_(t)
        return b, v

    (xb, xo), (db_, do), (yb, yo) = off(x), off(d), off(torch.zeros_like(x))
    dt = ops._DT[DT[dtype]]
    call("nsosx_layernorm", xo.data_ptr(), do.data_ptr(), w.data_ptr(), None, n, dim, 1e-5, dt, do.data_ptr(),
         yo.data_ptr(), dt, None, None, ops._stream())
    assert torch.equal(do, res) and torch.equal(yo, y) and torch.equal(xo, x)
    for b in (xb, db_, yb):  # nothing before or behind the rows
        assert b[0] == 7.0 and (b[1 + n * dim:] == 7.0).all()
    dy, _ = rows(rng, n, dim, dtype, dev, 0.01)
    want = ops.layernorm_backward(dy, res, mean, rstd, w, dresidual=d)
    (_, dyo), (gb, go) = off(dy), off(d)
    got = ops.layernorm_backward(dyo, do, mean, rstd, w, dresidual=go)
    assert all(torch.equal(got[k], want[k]) for k in want)
    ws = torch.empty(int(ops.lib().nsosx_layernorm_backward_workspace(n, dim)), dtype=torch.uint8, device=dev)
    call("nsosx_layernorm_backward", dyo.data_ptr(), dt, do.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
         w.data_ptr(), go.data_ptr(), n, dim, dt, go.data_ptr(), None, None, ws.data_ptr(), ops._stream())
    assert torch.equal(go, want["dx"]) and gb[0] == 7.0 and (gb[1 + n * dim:] == 7.0).all()


def test_values(dev):
    """Constant rows (variance 0), a large offset, and rows that are not finite by themselves."""
    dim = 300
    x = torch.ones((4, dim), device=dev)
    x[1] = 1e4 + torch.arange(dim, device=dev) % 3
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    w = torch.full((dim,), 2.0, device=dev)
    b = torch.full((dim,), 0.5, device=dev)
    y, mean, rstd = ops.layernorm(x, w, b, want_stats=True)
    assert torch.equal(y[0], torch.full((dim,), 0.5, device=dev))
    want, *_, lim, _, _ = ref.layernorm(x[1:2].double().cpu().numpy(), w.double().cpu().numpy(),
                                        b.double().cpu().numpy(), 1e-5)
    near(y[1:2], want, lim)
    assert torch.isnan(y[2:]).all(1).all()
    ok = ops.layernorm_backward(torch.ones_like(x), x, mean, rstd, w)
    assert torch.isfinite(ok["dx"][:2]).all() and torch.isnan(ok["dx"][2:]).any(1).all()


def test_no_rows(dev):
    x = torch.empty((0, 40), device=dev)
    y, mean, rstd = ops.layernorm(x, want_stats=True)
    assert y.shape == (0, 40)
    r = ops.layernorm_backward(x, x, mean, rstd)
    assert r["dx"].shape == (0, 40) and not r["dweight"].any() and not r["dbias"].any()


def test_offsets_past_32_bits(dev):
    """Rows behind the first 2^32 bytes (and 2^31 elements) of a buffer."""
    dim, n = 8192, (1 << 18) + 5
    x = torch.zeros((n, dim), dtype=torch.bfloat16, device=dev)
    tail = torch.randn((5, dim), device=dev).to(torch.bfloat16)
    x[-5:] = tail
    y, mean, rstd = ops.layernorm(x, want_stats=True)
    wy, wm, wr = ops.layernorm(tail, want_stats=True)
    assert torch.equal(y[-5:], wy) and torch.equal(mean[-5:], wm) and torch.equal(rstd[-5:], wr)
    assert not y[:-5].any()
    dx = ops.layernorm_backward(x, x, mean, rstd, want_params=False)["dx"]
    assert torch.equal(dx[-5:], ops.layernorm_backward(tail, tail, wm, wr, want_params=False)["dx"])


def test_streams_and_graphs(dev):
    rng = np.random.default_rng(9)
    x, _ = rows(rng, 700, 1000, "bf16", dev)
    d, _ = rows(rng, 700, 1000, "bf16", dev)
    w, _ = vec(rng, 1000, dev, 1.0)

    def both():
        res, y, mean, rstd = ops.add_layernorm(x, d, w, want_stats=True)
        r = ops.layernorm_backward(y, res, mean, rstd, w, dresidual=d)
        return [res, y, *r.values()]

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
        for t in out:
            t.fill_(float("nan"))
        ops.layernorm(torch.randn((3000, 500), device=dev))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
