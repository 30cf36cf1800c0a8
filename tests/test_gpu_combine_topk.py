"""The top-k combine and its gradients against 64-bit sums: odd widths, unaligned rows, padding
entries, rows no slot holds."""
import numpy as np
import pytest
import torch

from reimagined_amd import ops
from reimagined_amd._lib import call

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def make(dev, rows, k, dim, dtype, pad, seed=0):
    rng = np.random.default_rng([rows, k, dim, seed])
    slots = rows * k
    order = rng.permutation(slots).reshape(rows, k)
    if pad:  # dropped entries: their slots are the last ones, as a routing leaves them
        drop = rng.random((rows, k)) < 0.3
        slot = np.full((rows, k), -1)
        slot[~drop] = rng.permutation(int((~drop).sum()))
    else:
        slot = order
    y = torch.from_numpy(rng.normal(0, 1, (slots, dim)).astype(np.float32)).to(dtype)
    w = torch.from_numpy(rng.random((rows, k)).astype(np.float32))
    perm = np.full(slots, -1, np.int32)
    for r in range(rows):
        for i in range(k):
            if slot[r, i] >= 0:
                perm[slot[r, i]] = r
    return (y.to(dev), torch.from_numpy(slot.astype(np.int32)).to(dev), w.to(dev),
            torch.from_numpy(perm).to(dev), slot)


def forward64(y, slot, w):
    y = y.double().cpu().numpy()
    w = w.double().cpu().numpy() * (slot >= 0)
    rows = y[np.maximum(slot, 0)]
    return (rows * w[:, :, None]).sum(1), (np.abs(rows) * np.abs(w)[:, :, None]).sum(1)


SIZES = [(1, 1, 1), (1, 8, 4096), (3, 2, 7), (50, 4, 64), (33, 16, 520), (300, 2, 1024), (70, 6, 1001),
         (9, 3, 2056)]


@pytest.mark.parametrize("rows,k,dim", SIZES)
@pytest.mark.parametrize("idt", [F32, BF16])
@pytest.mark.parametrize("odt", [F32, BF16])
@pytest.mark.parametrize("pad", [False, True])
def test_combine(dev, rows, k, dim, idt, odt, pad):
    y, slot_t, w, _, slot = make(dev, rows, k, dim, idt, pad)
    got = ops.moe_combine_topk(y, slot_t, w, out_dtype=odt)
    assert got.dtype == odt
    want, mag = forward64(y, slot, w)
    # k fused steps, each half a step of a partial sum below `mag`, then the output's rounding
    lim = k * 2.0**-24 * mag + torch.finfo(odt).eps / 2 * np.abs(want) * (1 + 2.0**-8)
    assert (np.abs(got.double().cpu().numpy() - want) <= lim).all()


@pytest.mark.parametrize("rows,k,dim", SIZES)
@pytest.mark.parametrize("edt", [F32, BF16])
@pytest.mark.parametrize("ddt", [F32, BF16])
@pytest.mark.parametrize("pad", [False, True])
@pytest.mark.parametrize("with_perm", [False, True])
def test_backward(dev, rows, k, dim, edt, ddt, pad, with_perm):
    y, slot_t, w, perm, slot = make(dev, rows, k, dim, edt, pad)
    dout = torch.randn(rows, dim, device=dev, generator=torch.Generator(dev).manual_seed(dim)).to(ddt)
    de, dw = ops.moe_combine_topk_backward(dout, y, slot_t, w, perm=perm if with_perm else None)
    assert de.dtype == edt and dw.dtype == F32
    d = dout.double().cpu().numpy()
    y64, w64 = y.double().cpu().numpy(), w.double().cpu().numpy()
    want = np.zeros_like(y64)
    want_w = np.zeros((rows, k))
    mag = np.zeros((rows, k))
    for r in range(rows):
        for i in range(k):
            if slot[r, i] >= 0:
                want[slot[r, i]] = w64[r, i] * d[r]
                want_w[r, i] = y64[slot[r, i]] @ d[r]
                mag[r, i] = np.abs(y64[slot[r, i]]) @ np.abs(d[r])
    err = np.abs(de.double().cpu().numpy() - want)
    # one product rounded to 32 bits, then to the type
    assert (err <= (2.0**-24 + torch.finfo(edt).eps / 2 * (1 + 2.0**-23)) * np.abs(want) + 1e-40).all()
    # fused steps: dim / 64 in a lane at most (one element a step), 6 + 3 additions across
    steps = dim / 64 + 17
    assert (np.abs(dw.double().cpu().numpy() - want_w) <= steps * 2.0**-24 * mag).all()


def test_gradients_against_differences(dev):
    """out . dout moves by dw along a weight and by dexpert along an expert's element."""
    y, slot_t, w, perm, slot = make(dev, 6, 3, 24, F32, True, seed=4)
    dout = torch.randn(6, 24, device=dev, generator=torch.Generator(dev).manual_seed(1))
    de, dw = ops.moe_combine_topk_backward(dout, y, slot_t, w, perm=perm)

    def loss(yv, wv):
        w0 = wv * (slot >= 0)
        return ((yv[np.maximum(slot, 0)] * w0[:, :, None]).sum(1) * dout.double().cpu().numpy()).sum()

    y64, w64 = y.double().cpu().numpy(), w.double().cpu().numpy()
    h = 1e-3  # the loss is bilinear: central differences are exact to rounding
    for r in range(6):
        for i in range(3):
            up, dn = w64.copy(), w64.copy()
            up[r, i] += h
            dn[r, i] -= h
            assert abs((loss(y64, up) - loss(y64, dn)) / (2 * h) - dw[r, i].item()) < 1e-5
    for s, d in [(0, 0), (3, 7), (5, 23), (17, 4)]:
        up, dn = y64.copy(), y64.copy()
        up[s, d] += h
        dn[s, d] -= h
        assert abs((loss(up, w64) - loss(dn, w64)) / (2 * h) - de[s, d].item()) < 1e-5


def test_unaligned_rows_and_slots_past_the_end(dev):
    """Rows that start at any element, and slots no expert row exists for, which add nothing and
    are not written."""
    rows, k, dim, slots = 5, 2, 64, 10
    flat = torch.randn(slots * dim + 1, device=dev, generator=torch.Generator(dev).manual_seed(2)).to(BF16)
    y = flat[1:].view(slots, dim)
    slot = torch.tensor([[0, 9], [10, 1], [2, 1000000], [-5, 3], [4, 5]], dtype=torch.int32, device=dev)
    w = torch.rand(rows, k, device=dev, generator=torch.Generator(dev).manual_seed(3))
    got = ops.moe_combine_topk(y, slot, w)
    sl = slot.cpu().numpy()
    sl[(sl < 0) | (sl >= slots)] = -1
    want, mag = forward64(y, sl, w)
    assert (np.abs(got.double().cpu().numpy() - want) <= k * 2.0**-24 * mag + 2.0**-24 * np.abs(want)).all()
    guard = torch.full((slots + 8, dim), 7.0, device=dev, dtype=BF16)
    dw = torch.empty(rows, k, device=dev)
    dout = torch.randn(rows, dim, device=dev, generator=torch.Generator(dev).manual_seed(4))
    call("nsosx_moe_combine_topk_backward", dout.data_ptr(), 0, y.data_ptr(), 1, slot.data_ptr(),
         w.data_ptr(), None, rows, slots, k, dim, guard.data_ptr(), dw.data_ptr(), ops._stream())
    assert (guard[slots:] == 7.0).all() and (guard[6:9] == 7.0).all()
    assert dw[1, 0] == 0 and dw[2, 1] == 0 and dw[3, 0] == 0
