"""Refusals of layer norm, the gated recurrence and the balance loss (CPU only): the wrappers on CPU
tensors, the C entries on placeholder addresses that no check dereferences."""
import pytest
import torch

from reimagined_amd import _lib, ops

P = 1 << 30  # placeholder addresses, never dereferenced, far apart
Q, R, S, T = P * 3, P * 5, P * 7, P * 9


def refused(fn, *args, status=1):
    lib = _lib.lib()
    assert getattr(lib, fn)(*args) == status, lib.nsosx_last_error().decode()
    return lib.nsosx_last_error().decode()


# ---- layer norm -------------------------------------------------------------------

def ln(x=P, delta=None, rows=4, dim=8, eps=1e-5, dt=0, sum=None, y=Q, odt=0, mean=None, rstd=None):
    return (x, delta, None, None, rows, dim, eps, dt, sum, y, odt, mean, rstd, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(rows=-1), "rows >= 0"), (dict(dim=0), "dim > 0"),
    (dict(dt=2), "dtype"), (dict(odt=-1), "dtype"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(delta=R), "together"), (dict(sum=R), "together"),
    (dict(mean=R), "together"), (dict(y=P), "overlaps"), (dict(y=P + 124), "overlaps"),
    (dict(delta=R, sum=S, y=S), "overlaps"), (dict(delta=R, sum=S, y=R), "overlaps"),
    (dict(delta=R, sum=P + 4), "cross"), (dict(delta=R, sum=R + 4), "cross"),
])
def test_layernorm_refusals(kw, text):
    assert text in refused("nsosx_layernorm", *ln(**kw))


def test_layernorm_too_large():
    assert "too large" in refused("nsosx_layernorm", *ln(rows=1, dim=2**30 + 1, y=P * 64), status=2)
    assert "too large" in refused("nsosx_layernorm", *ln(rows=2**28, dim=300, y=P * 4096), status=2)
    assert _lib.lib().nsosx_layernorm_backward_workspace(4, 0) == 0


def lnb(dy=P, gdt=0, x=Q, mean=R, rstd=R, dres=None, rows=4, dim=8, dt=0, dx=S, dw=T, db=T, ws=T):
    return (dy, gdt, x, mean, rstd, None, dres, rows, dim, dt, dx, dw, db, ws, None)


@pytest.mark.parametrize("kw,text", [
    (dict(dy=None), "null"), (dict(x=None), "null"), (dict(mean=None), "null"), (dict(rstd=None), "null"),
    (dict(dx=None), "null"), (dict(ws=None), "null"), (dict(ws=None, dw=None), "null"), (dict(rows=-1), "rows"),
    (dict(dim=0), "dim"), (dict(dt=2), "dtype"), (dict(gdt=2), "dtype"), (dict(dx=P), "overlaps"),
    (dict(dx=Q + 4), "overlaps"), (dict(dres=S + 4), "overlaps"),
])
def test_layernorm_backward_refusals(kw, text):
    assert text in refused("nsosx_layernorm_backward", *lnb(**kw))


def test_layernorm_wrappers():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="device tensor"):
        ops.layernorm(x)
    with pytest.raises(ValueError, match="rows, dim"):
        ops.layernorm(torch.zeros(8))
    with pytest.raises(ValueError, match="dtype"):
        ops.layernorm(x.half())
    with pytest.raises(ValueError, match="out_dtype"):
        ops.layernorm(x, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensor"):
        ops.add_layernorm(x, x)
    with pytest.raises(ValueError, match="device tensor"):
        ops.layernorm_backward(x, x, x[:, 0], x[:, 0])


# ---- gated recurrence ---------------------------------------------------------------

def rec(x=P, xs=8, rg=2 * P, rs=8, ig=Q, igs=8, lam=R, rate=8.0, cu=R, s=2, t=4, d=8, dt=0, h0=None, y=S, ys=8,
        final=None, carry=None, ws=T):
    return (x, xs, rg, rs, ig, igs, lam, rate, cu, s, t, d, dt, h0, 1, y, ys, final, carry, ws, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(rg=None), "null"), (dict(ig=None), "null"), (dict(lam=None), "null"),
    (dict(cu=None), "null"), (dict(y=None), "null"), (dict(ws=None), "null"), (dict(s=-1), "sequences"),
    (dict(t=-1), "tokens"), (dict(d=0), "dim"), (dict(dt=2), "dtype"), (dict(rate=0.0), "rate"),
    (dict(rate=-1.0), "rate"), (dict(rate=float("inf")), "rate"), (dict(rate=float("nan")), "rate"),
    (dict(xs=7), "stride"), (dict(rs=7), "stride"), (dict(igs=0), "stride"), (dict(ys=7), "stride"),
    (dict(y=P), "overlaps"), (dict(y=2 * P + 4), "overlaps"), (dict(y=Q + 3 * 32 + 28), "overlaps"),
    (dict(x=P, xs=16, y=P + 28, ys=16), "overlaps"), (dict(x=P, xs=16, y=P + 32, ys=24), "overlaps"),
    (dict(h0=T, final=T), "overlaps"), (dict(h0=T, final=T + 4), "overlaps"),
])
def test_recurrence_refusals(kw, text):
    assert text in refused("nsosx_gated_recurrence", *rec(**kw))


def test_recurrence_too_large():
    assert "too large" in refused("nsosx_gated_recurrence", *rec(d=2**30 + 1, xs=2**31, rs=2**31, igs=2**31,
                                                                 ys=2**31), status=2)
    assert "too large" in refused("nsosx_gated_recurrence", *rec(s=2**20, d=8192, xs=8192, rs=8192, igs=8192,
                                                                 ys=8192), status=2)
    assert "too large" in refused("nsosx_gated_recurrence_backward", *recb(t=2**31 - 1, d=2**20), status=2)
    assert _lib.lib().nsosx_gated_recurrence_workspace(0, 8) == 0


def recb(dy=P, dys=8, x=2 * P, rg=3 * P, ig=4 * P, lam=R, cu=R, s=2, t=4, d=8, dt=0, h0=None, carry=T, dfinal=None,
         dx=10 * P, dxs=8, drg=11 * P, drs=8, dig=12 * P, dis=8, dlam=13 * P, dinit=None, ws=14 * P, rate=8.0):
    return (dy, dys, x, max(8, d), rg, max(8, d), ig, max(8, d), lam, rate, cu, s, t, d, dt, h0, carry, dfinal, 1,
            dx, dxs, drg, drs, dig, dis, dlam, dinit, ws, None)


@pytest.mark.parametrize("kw,text", [
    (dict(dy=None), "null"), (dict(x=None), "null"), (dict(rg=None), "null"), (dict(ig=None), "null"),
    (dict(lam=None), "null"), (dict(cu=None), "null"), (dict(carry=None), "null"), (dict(dx=None), "null"),
    (dict(drg=None), "null"), (dict(dig=None), "null"), (dict(dlam=None), "null"), (dict(ws=None), "null"),
    (dict(s=-1), "sequences"), (dict(t=-1), "tokens"), (dict(d=0), "dim"), (dict(dt=3), "dtype"),
    (dict(rate=0.0), "rate"), (dict(dys=7), "stride"), (dict(dxs=7), "stride"), (dict(drs=7), "stride"),
    (dict(dis=7), "stride"), (dict(dx=P), "overlaps"), (dict(dig=3 * P + 4), "overlaps"),
    (dict(drg=10 * P), "overlap"), (dict(dxs=24, drg=10 * P + 32, drs=24, dig=10 * P + 60, dis=24), "overlap"),
    (dict(dfinal=15 * P, dinit=15 * P), "overlaps"), (dict(h0=15 * P, dinit=15 * P + 4), "overlaps"),
])
def test_recurrence_backward_refusals(kw, text):
    assert text in refused("nsosx_gated_recurrence_backward", *recb(**kw))


def step(x=P, xs=8, rg=2 * P, ig=Q, lam=R, rate=8.0, rows=4, d=8, dt=0, state=S, out=S, y=T, ys=8):
    return (x, xs, rg, max(8, d), ig, max(8, d), lam, rate, rows, d, dt, state, out, y, ys, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(lam=None), "null"), (dict(state=None), "null"), (dict(out=None), "null"),
    (dict(y=None), "null"), (dict(rows=-1), "tokens"), (dict(d=0), "dim"), (dict(dt=2), "dtype"),
    (dict(rate=-2.0), "rate"), (dict(xs=7), "stride"), (dict(ys=7), "stride"), (dict(out=S + 4), "cross"),
    (dict(y=P), "overlaps"),
])
def test_step_refusals(kw, text):
    assert text in refused("nsosx_gated_recurrence_step", *step(**kw))


def test_recurrence_wrappers():
    x, lam, cu = torch.zeros(4, 8), torch.zeros(8), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        ops.gated_recurrence(x, x, x, lam, cu)
    with pytest.raises(ValueError, match="tokens, dim"):
        ops.gated_recurrence(x[0], x[0], x[0], lam, cu)
    with pytest.raises(ValueError, match="dtype"):
        ops.gated_recurrence(x.half(), x, x, lam, cu)
    with pytest.raises(ValueError, match="device tensor"):
        ops.gated_recurrence_step(x, x, x, lam, x)
    with pytest.raises(ValueError, match="device tensor"):
        ops.gated_recurrence_backward(x, x, x, x, lam, cu, x)


# ---- balance loss ---------------------------------------------------------------------

def bal(x=P, dt=0, stride=8, sel=Q, rows=4, e=8, k=2, cu=None, s=1, loss=R, counts=R, tokens=R, mean=R, ws=R):
    return (x, dt, stride, sel, None, rows, e, k, 0, cu, s, loss, counts, tokens, mean, ws, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(sel=None), "null"), (dict(loss=None), "null"), (dict(counts=None), "null"),
    (dict(tokens=None), "null"), (dict(mean=None), "null"), (dict(ws=None), "null"), (dict(rows=-1), "rows"),
    (dict(e=0), "E <= 512"), (dict(e=513, stride=513), "E <= 512"), (dict(k=0), "k"), (dict(k=9), "k"),
    (dict(k=17, e=64, stride=64), "k <= 16"), (dict(dt=2), "dtype"), (dict(s=2), "cu_seqlens"),
    (dict(cu=R, s=-1), "sequences"), (dict(stride=7), "stride"),
])
def test_balance_refusals(kw, text):
    assert text in refused("nsosx_moe_balance_loss", *bal(**kw))


def balb(x=P, dt=0, stride=8, counts=Q, tokens=Q, rows=4, e=8, k=2, cu=None, s=1, add=None, out=S):
    return (x, dt, stride, counts, tokens, None, rows, e, k, 0, cu, s, 1.0, None, add, out, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(counts=None), "null"), (dict(tokens=None), "null"), (dict(out=None), "null"),
    (dict(e=513, stride=513), "E <= 512"), (dict(k=9), "k"), (dict(dt=2), "dtype"), (dict(s=0), "cu_seqlens"),
    (dict(stride=7), "stride"), (dict(out=P), "overlaps"), (dict(out=Q), "overlaps"), (dict(add=S + 4), "overlaps"),
])
def test_balance_backward_refusals(kw, text):
    assert text in refused("nsosx_moe_balance_loss_backward", *balb(**kw))


def test_balance_too_large():
    assert "too large" in refused("nsosx_moe_balance_loss", *bal(rows=2**28), status=2)


def test_balance_wrappers():
    x, sel = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        ops.moe_balance_loss(x, sel)
    with pytest.raises(ValueError, match="device tensor"):
        ops.moe_balance_loss_backward(x, sel, sel, 2)


def test_recurrence_bounds():
    x, lam = torch.zeros(4, 8), torch.zeros(8)
    for cu in (None, torch.zeros((2, 2), dtype=torch.int32), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="cu_seqlens must be"):
            ops.gated_recurrence(x, x, x, lam, cu)
        with pytest.raises(ValueError, match="cu_seqlens must be"):
            ops.gated_recurrence_backward(x, x, x, x, lam, cu, torch.zeros(1, 8))
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for bad in (torch.zeros(()), torch.zeros(4), torch.zeros(2, 2, 8), torch.zeros(4, 0)):
        with pytest.raises(ValueError, match="tokens, dim"):
            ops.gated_recurrence(bad, x, x, lam, cu)
        with pytest.raises(ValueError, match="tokens, dim"):
            ops.gated_recurrence_backward(x, bad, x, x, lam, cu, torch.zeros(1, 8))


def test_layer_refusals():
    from reimagined_amd.layers import RecurrentLayer
    p = lambda **kw: {"w_in": torch.zeros(96, 48), "w_out": torch.zeros(48, 32), "lam": torch.zeros(32), **kw}
    for bad in (dict(w_in=torch.zeros(95, 48)), dict(w_out=torch.zeros(32, 48)), dict(lam=torch.zeros(31)),
                dict(w_in=torch.zeros(96, 40), w_out=torch.zeros(40, 32)), dict(b_in=torch.zeros(32))):
        with pytest.raises(ValueError, match="RecurrentLayer"):
            RecurrentLayer(p(**bad), "cpu")
    with pytest.raises(ValueError, match="train=True"):
        RecurrentLayer.backward(None, {"residual": None, "out": None, "final_state": None}, None)
