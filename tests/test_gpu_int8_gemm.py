"""int8 products, one matrix and grouped, bit for bit: the sums are exact integers and the affine
is one rounding to 32 bits at the conversion, each product and the sum, which numpy's float32
does alike."""
import numpy as np
import pytest
import torch

from reimagined_amd import ops
from reimagined_amd._lib import call

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def affine(acc, s, ws, bias, sqrelu):
    v = acc.astype(np.float32) * s[:, None] * ws[None, :]
    if bias is not None:
        v = v + bias[None, :]
    if sqrelu:
        v = np.where(v < 0, np.float32(0), v)
        v = v * v
    return v


def product(q, s, w, ws, bias=None, sqrelu=False):
    """q, w int8 -> float32; the integer sums in float64, exact below 2^53."""
    return affine(q.astype(np.float64) @ w.astype(np.float64).T, s, ws, bias, sqrelu)


def same(got, want, dtype):
    assert got.dtype == dtype
    want = torch.from_numpy(np.ascontiguousarray(want)).to(dtype)
    assert torch.equal(got.cpu(), want), (got.cpu().float() - want.float()).abs().max()


def operands(rng, m, k, n):
    return (rng.integers(-127, 128, (m, k)).astype(np.int8), rng.uniform(1e-3, 2e-2, m).astype(np.float32),
            rng.integers(-127, 128, (n, k)).astype(np.int8), rng.uniform(1e-4, 2e-3, n).astype(np.float32),
            rng.normal(0, 1, n).astype(np.float32))


def t(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


@pytest.mark.parametrize("k", [1, 15, 16, 17, 64, 100, 127, 128, 144, 1000, 2009, 4096])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 33), (2, 256), (16, 17), (17, 64), (33, 130), (64, 5),
                                 (70, 300), (129, 127), (300, 520), (257, 256), (600, 48)])
def test_sizes(dev, m, k, n):
    rng = np.random.default_rng([m, k, n])
    q, s, w, ws, b = operands(rng, m, k, n)
    dq, dsc, dw, dws, db = (t(a, dev) for a in (q, s, w, ws, b))
    same(ops.int8_gemm(dq, dsc, dw, dws, bias=db), product(q, s, w, ws, b), F32)
    same(ops.int8_gemm(dq, dsc, dw, dws, out_dtype=BF16), product(q, s, w, ws), BF16)


@pytest.mark.parametrize("m,k,n", [(1024, 1024, 1024), (513, 2048, 4096), (2000, 640, 1536),
                                   (4096, 256, 2056), (1100, 1040, 2049)])
def test_large_tiles(dev, m, k, n):
    rng = np.random.default_rng([m, k, n])
    q, s, w, ws, b = operands(rng, m, k, n)
    dq, dsc, dw, dws, db = (t(a, dev) for a in (q, s, w, ws, b))
    want = product(q, s, w, ws, b)
    same(ops.int8_gemm(dq, dsc, dw, dws, bias=db), want, F32)
    same(ops.int8_gemm(dq, dsc, dw, dws, bias=db, out_dtype=BF16), want, BF16)


@pytest.mark.parametrize("m", [1, 40, 200])
@pytest.mark.parametrize("off", [1, 4, 8])
def test_unaligned_operands(dev, m, off):
    """Codes, weights and outputs that start at any byte / element."""
    rng = np.random.default_rng(off)
    k, n = 192, 136
    q, s, w, ws, b = operands(rng, m, k, n)
    fq = torch.zeros(m * k + 16, dtype=torch.int8, device=dev)
    fw = torch.zeros(n * k + 16, dtype=torch.int8, device=dev)
    fq[off:off + m * k] = t(q, dev).view(-1)
    fw[off:off + n * k] = t(w, dev).view(-1)
    fy = torch.full((m * n + 16,), 9.0, dtype=BF16, device=dev)
    y = fy[off:off + m * n]
    ds, dws = t(s, dev), t(ws, dev)
    call("nsosx_int8_gemm", fq.data_ptr() + off, ds.data_ptr(), fw.data_ptr() + off, dws.data_ptr(), None, m, k, n, y.data_ptr(), 1, ops._stream())
    torch.cuda.synchronize()
    same(y.view(m, n), product(q, s, w, ws), BF16)
    assert (fy[:off] == 9).all() and (fy[off + m * n:] == 9).all()


@pytest.mark.parametrize("m", [1, 17, 150, 300])
def test_longest_k_and_extreme_codes(dev, m):
    """K = 131071 of -128 * -128: the largest sum, 2^31 - 16384."""
    k, n = 131071, 20
    q = np.full((m, k), -128, np.int8)
    w = np.full((n, k), -128, np.int8)
    w[1::2] = 127
    s, ws = np.ones(m, np.float32), np.full(n, 0.5, np.float32)
    got = ops.int8_gemm(t(q, dev), t(s, dev), t(w, dev), t(ws, dev)).cpu().numpy()
    row = np.float32(np.where(np.arange(n) % 2, -128 * 127 * k, 128 * 128 * k).astype(np.float64)) * np.float32(0.5)
    assert (got == row[None]).all()


def test_nan_and_infinite_scales(dev):
    rng = np.random.default_rng(1)
    for m in (3, 200):
        q, s, w, ws, b = operands(rng, m, 64, 70)
        s[1], ws[4], b[6] = np.nan, np.inf, np.nan
        got = ops.int8_gemm(t(q, dev), t(s, dev), t(w, dev), t(ws, dev), bias=t(b, dev)).cpu().numpy()
        want = product(q, s, w, ws, b)
        np.testing.assert_array_equal(got, want)  # NaN where NaN
        off = np.array([0, m], np.int32)
        got = ops.grouped_int8_gemm(t(q, dev), t(s, dev), t(w[None], dev), t(ws[None], dev), t(off, dev),
                                    bias=t(b[None], dev), squared_relu=True).cpu().numpy()
        np.testing.assert_array_equal(got, product(q, s, w, ws, b, True))


def test_offsets_past_32_bits(dev):
    """Weights, and outputs, of more than 2^31 elements."""
    k, n = 65536, 33000
    g = torch.Generator(dev).manual_seed(1)
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=dev, generator=g)
    q = torch.randint(-127, 128, (150, k), dtype=torch.int8, device=dev, generator=g)
    ws, s = torch.full((n,), 1e-3, device=dev), torch.full((150,), 1e-2, device=dev)
    want = product(q.cpu().numpy(), s.cpu().numpy(), w[-20:].cpu().numpy(), ws[-20:].cpu().numpy())
    for m in (1, 150):
        got = ops.int8_gemm(q[:m].contiguous(), s[:m].contiguous(), w, ws)
        same(got[:, -20:].contiguous(), want[:m], F32)
    del w, got
    m, n, k = 70000, 33000, 32
    q = torch.randint(-127, 128, (m, k), dtype=torch.int8, device=dev, generator=g)
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=dev, generator=g)
    s, ws = torch.full((m,), 1e-2, device=dev), torch.full((n,), 1e-3, device=dev)
    got = ops.int8_gemm(q, s, w, ws, out_dtype=BF16)
    for rows in (slice(0, 5), slice(m - 300, m)):
        want = product(q[rows].cpu().numpy(), s[rows].cpu().numpy(), w.cpu().numpy(), ws.cpu().numpy())
        same(got[rows], want, BF16)


# ---- grouped -------------------------------------------------------------------------

def segments(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def grouped_ref(q, s, w, ws, off, perm, bias, sqrelu):
    slots = off[-1]
    at = np.arange(slots) if perm is None else perm[:slots]
    out = np.zeros((slots, w.shape[1]), np.float32)
    for e in range(len(w)):
        r = at[off[e]:off[e + 1]]
        if len(r):
            out[off[e]:off[e + 1]] = product(q[r], s[r], w[e], ws[e], None if bias is None else bias[e], sqrelu)
    return out


COUNTS = [[1], [0, 0, 3], [5, 0, 17, 64, 0, 1], [130, 128, 0, 127, 1], [16] * 40, [0] * 70 + [9],
          [700, 3, 0, 600], [33, 250, 40, 129, 0, 300], [2000, 0, 0, 0]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("k,n", [(64, 48), (128, 256), (100, 33), (272, 520)])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped(dev, counts, k, n, gather):
    rng = np.random.default_rng([len(counts), sum(counts), k, n])
    off = segments(counts)
    slots, e = int(off[-1]), len(counts)
    rows = max(1, slots // 2 + 3) if gather else slots
    q, s, _, _, _ = operands(rng, rows, k, 1)
    w = rng.integers(-127, 128, (e, n, k)).astype(np.int8)
    ws = rng.uniform(1e-4, 2e-3, (e, n)).astype(np.float32)
    b = rng.normal(0, 1, (e, n)).astype(np.float32)
    perm = rng.integers(0, rows, slots).astype(np.int32) if gather else None
    args = [t(a, dev) for a in (q, s, w, ws, off)]
    pt = None if perm is None else t(perm, dev)
    same(ops.grouped_int8_gemm(*args, perm=pt, bias=t(b, dev), squared_relu=True),
         grouped_ref(q, s, w, ws, off, perm, b, True), F32)
    same(ops.grouped_int8_gemm(*args, perm=pt, out_dtype=BF16),
         grouped_ref(q, s, w, ws, off, perm, None, False), BF16)


@pytest.mark.parametrize("slots", [50, 900])
def test_rows_past_the_last_segment_are_left(dev, slots):
    """Padding: offsets[E] below the slots, perm -1 behind it."""
    rng = np.random.default_rng(slots)
    counts = [slots // 3, 0, slots // 4]
    off = segments(counts)
    k, n, rows = 96, 72, 40
    q, s, _, _, _ = operands(rng, rows, k, 1)
    w = rng.integers(-127, 128, (3, n, k)).astype(np.int8)
    ws = rng.uniform(1e-4, 2e-3, (3, n)).astype(np.float32)
    perm = np.full(slots, -1, np.int32)
    perm[:off[-1]] = rng.integers(0, rows, off[-1])
    y = torch.full((slots, n), 9.0, device=dev)
    dv = [t(a, dev) for a in (q, s, w, ws, off, perm)]
    call("nsosx_grouped_int8_gemm", dv[0].data_ptr(), dv[1].data_ptr(), rows, dv[2].data_ptr(),
         dv[3].data_ptr(), None, dv[4].data_ptr(), dv[5].data_ptr(), slots, 3, k, n, 0, y.data_ptr(), 0,
         ops._stream())
    same(y[:off[-1]], grouped_ref(q, s, w, ws, off, perm, None, False), F32)
    assert (y[off[-1]:] == 9).all()


def test_many_experts_few_rows(dev):
    """1024 experts, three of them with a row."""
    rng = np.random.default_rng(2)
    counts = np.zeros(1024, int)
    counts[[0, 511, 1023]] = 1
    off = segments(counts)
    q, s, _, _, _ = operands(rng, 3, 64, 1)
    w = rng.integers(-127, 128, (1024, 16, 64)).astype(np.int8)
    ws = rng.uniform(1e-4, 2e-3, (1024, 16)).astype(np.float32)
    got = ops.grouped_int8_gemm(*[t(a, dev) for a in (q, s, w, ws, off)])
    same(got, grouped_ref(q, s, w, ws, off, None, None, False), F32)
