"""Every tile of the int8 products, each on shapes that it takes by the library's own rule: whole and
partial steps of K, an odd and an even number of stages, ragged rows and outputs, rows that start
anywhere, both types, with and without a bias and the activation, nothing written outside.  Bit for
bit, as the sums are exact."""
import numpy as np
import pytest
import torch

from reimagined_amd import _lib, ops
from reimagined_amd._lib import call

from test_gpu_int8_gemm import affine, grouped_ref, operands, segments, t

F32, BF16 = torch.float32, torch.bfloat16

# rows, K, N, tile (the index that nsosx_int8_gemm_tile returns).  K in stages of 64 (tiles 0 to 3) or
# 128 (4 and 5): fewer than one, one, odd and even numbers of them, with and without a rest.
ALIGNED = [(5, 1040, 300, 0), (40, 4096, 130, 0), (150, 1040, 1030, 1), (90, 4096, 1530, 1),
           (129, 4096, 1536, 2), (77, 2064, 2050, 2), (77, 2064, 5125, 3), (150, 4096, 4101, 3),
           (400, 1040, 4096, 4), (1030, 640, 2056, 4), (500, 144, 4098, 4), (2000, 112, 2001, 4),
           (4095, 112, 4090, 5), (4090, 128, 4096, 5), (4081, 384, 4089, 5), (4090, 656, 4090, 5),
           (4090, 1040, 4096, 5), (4088, 1024, 4081, 5)]
ODD = [(5, 1041, 300, 0), (40, 4095, 130, 0), (150, 1041, 1030, 1), (33, 2009, 4096, 1), (77, 2009, 2050, 2),
       (129, 4095, 1536, 2), (77, 2009, 5125, 3), (150, 2009, 4096, 3), (400, 2009, 4096, 4),
       (1100, 401, 2049, 4), (2048, 145, 4096, 4), (2000, 127, 2000, 4), (2000, 15, 2000, 4), (2000, 385, 2003, 4)]
# slots, experts, K, N, tile
GROUPED = [(64, 8, 1040, 300, 0), (520, 26, 2064, 130, 1), (130, 3, 2064, 1100, 2), (150, 2, 2064, 4100, 2),
           (100, 5, 2064, 2100, 3), (300, 17, 2064, 520, 3), (300, 4, 1040, 2050, 4),
           (1000, 5, 400, 2050, 4), (3000, 5, 112, 2056, 4), (2000, 8, 144, 4100, 5), (3400, 3, 384, 4089, 5),
           (3500, 2, 656, 4090, 5), (3600, 1, 656, 4090, 5), (3000, 4, 1040, 4090, 5)]
GROUPED_ODD = [(64, 8, 1041, 300, 0), (520, 21, 401, 130, 1), (130, 3, 2009, 1100, 2), (150, 16, 2009, 520, 2),
               (300, 17, 2009, 520, 3), (64, 3, 1041, 2100, 3), (300, 4, 1041, 2050, 4),
               (3000, 5, 401, 2050, 4), (1000, 5, 15, 2050, 4)]


def tile(rows, k, n, experts=0, aligned=1):
    return _lib.lib().nsosx_int8_gemm_tile(rows, k, n, experts, aligned)


def test_the_shapes_take_their_tiles():
    """(The rule may be fitted again: the shapes below then have to follow it.)"""
    assert [s for s in ALIGNED + ODD if tile(*s[:3]) != s[3]] == []
    assert [s for s in GROUPED + GROUPED_ODD if tile(s[0], s[2], s[3], s[1]) != s[4]] == []
    for cases in (ALIGNED, GROUPED):
        assert {s[-1] for s in cases} == {0, 1, 2, 3, 4, 5}
    for cases in (ODD, GROUPED_ODD):
        assert {s[-1] for s in cases} == {0, 1, 2, 3, 4}
    assert tile(4090, 656, 4090, aligned=0) == 4  # rows on any byte have no 256 x 256


@pytest.mark.parametrize("args", [(0, 16, 16, 0, 1), (1, 0, 16, 0, 1), (1, 131072, 16, 0, 1), (1, 16, 0, 0, 1),
                                  (1, 16, 16, -1, 1), (1, 16, 16, 1025, 1), (2**30 + 1, 16, 1, 0, 1),
                                  (1, 16, 2**30 + 1, 3, 1), (2**20, 16, 2**20, 0, 1), (2**20, 16, 2**20, 3, 1)])
def test_no_tile_for_refused_sizes(args):
    assert tile(*args) == -1


class Guarded:
    """An output [rows, n] with other rows before and behind it; `at` elements past 16 bytes."""

    def __init__(self, dev, rows, n, dtype, at):
        self.size, self.at = rows * n, 64 + at
        self.all = torch.full((self.size + 128,), 9.0, dtype=dtype, device=dev)
        self.y = self.all[self.at:self.at + self.size].view(rows, n)

    def check(self, want, rows=None):
        """The first `rows` rows are `want`, all else is as it was."""
        rows = self.y.shape[0] if rows is None else rows
        want = torch.from_numpy(np.ascontiguousarray(want)).to(self.all.dtype)
        assert torch.equal(self.y[:rows].cpu(), want)
        assert (self.all[:self.at] == 9).all() and (self.all[self.at + rows * self.y.shape[1]:] == 9).all()


def on_byte(a, dev, off):
    """A device copy of an int8 array that starts `off` bytes past 16."""
    flat = torch.zeros(a.size + 32, dtype=torch.int8, device=dev)
    flat[off:off + a.size] = t(a, dev).view(-1)
    return flat[off:off + a.size].view(a.shape)


def run_matrix(dev, m, k, n, off):
    rng = np.random.default_rng([m, k, n])
    q, s, w, ws, b = operands(rng, m, k, n)
    acc = q.astype(np.float64) @ w.astype(np.float64).T
    dq, dw = on_byte(q, dev, off), on_byte(w, dev, off)
    ds, dws, db = (t(a, dev) for a in (s, ws, b))
    for bias in (None, b):
        want = affine(acc, s, ws, bias, False)
        for dtype, code in ((F32, 0), (BF16, 1)):
            for at in (0, 1):
                y = Guarded(dev, m, n, dtype, at)
                call("nsosx_int8_gemm", dq.data_ptr(), ds.data_ptr(), dw.data_ptr(), dws.data_ptr(),
                     None if bias is None else db.data_ptr(), m, k, n, y.y.data_ptr(), code, ops._stream())
                y.check(want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,kind", ALIGNED + ODD)
def test_matrix(dev, m, k, n, kind):
    assert tile(m, k, n) == kind
    run_matrix(dev, m, k, n, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,kind", [(40, 4096, 130, 0), (150, 1040, 1030, 1), (77, 2064, 2050, 2),
                                        (77, 2064, 5125, 3), (400, 1040, 4096, 4), (1500, 128, 2056, 4)])
@pytest.mark.parametrize("off", [1, 8])
def test_matrix_on_any_byte(dev, m, k, n, kind, off):
    assert tile(m, k, n, aligned=0) == kind
    run_matrix(dev, m, k, n, off)


@pytest.mark.gpu
@pytest.mark.parametrize("slots,e,k,n,kind", GROUPED + GROUPED_ODD)
@pytest.mark.parametrize("gather", [False, True])
def test_experts(dev, slots, e, k, n, kind, gather):
    """Uneven segments, an empty one where there are several, and slots behind the last."""
    assert tile(slots, k, n, e) == kind
    rng = np.random.default_rng([slots, e, k, n])
    share = rng.dirichlet(np.full(e, 2.0))
    if e > 2:
        share[1] = 0
    counts = (share * (slots - 3)).astype(int)
    off = segments(counts)
    used = int(off[-1])
    rows = slots // 2 + 3 if gather else slots
    q, s, _, _, _ = operands(rng, rows, k, 1)
    w = rng.integers(-127, 128, (e, n, k)).astype(np.int8)
    ws = rng.uniform(1e-4, 2e-3, (e, n)).astype(np.float32)
    b = rng.normal(0, 1, (e, n)).astype(np.float32)
    perm = None
    if gather:
        perm = np.full(slots, -1, np.int32)
        perm[:used] = rng.integers(0, rows, used)
    dq, ds, dw, dws, do, db = (t(a, dev) for a in (q, s, w, ws, off, b))
    dp = None if perm is None else t(perm, dev)
    for bias, sqrelu in ((None, 0), (b, 1), (b, 0), (None, 1)):
        want = grouped_ref(q, s, w, ws, off, perm, bias, bool(sqrelu))
        for dtype, code in ((F32, 0), (BF16, 1)):
            y = Guarded(dev, slots, n, dtype, sqrelu)
            call("nsosx_grouped_int8_gemm", dq.data_ptr(), ds.data_ptr(), rows, dw.data_ptr(), dws.data_ptr(),
                 None if bias is None else db.data_ptr(), do.data_ptr(), None if dp is None else dp.data_ptr(),
                 slots, e, k, n, sqrelu, y.y.data_ptr(), code, ops._stream())
            y.check(want, used)
