"""Refusals of scored routing, the top-k combine and the int8 products (CPU only): the wrappers
on CPU tensors, the C entries on placeholder addresses that no check dereferences."""
import pytest
import torch

from reimagined_amd import _lib, ops

P = 1 << 20  # a placeholder address, never dereferenced


def refused(fn, *args, status=1):
    lib = _lib.lib()
    assert getattr(lib, fn)(*args) == status, lib.nsosx_last_error().decode()
    return lib.nsosx_last_error().decode()


def route(logits=P, dt=0, stride=64, rows=4, e=64, k=2, groups=1, keep=1, best=1, w=P, sel=P, c=P, o=P,
          perm=P, slot=P, ws=P):
    return (logits, dt, stride, None, None, rows, e, k, 0, groups, keep, best, 1, 1.0, w, sel, c, o, perm,
            slot, ws, None)


@pytest.mark.parametrize("kw,text", [
    (dict(logits=None), "null"), (dict(w=None), "null"), (dict(sel=None), "null"),
    (dict(c=None), "null"), (dict(perm=None), "null"), (dict(ws=None), "null"),
    (dict(dt=2), "dtype"), (dict(rows=0), "rows > 0"), (dict(e=0, stride=1), "E <= 512"),
    (dict(e=513, stride=513), "E <= 512"), (dict(k=0), "0 < k"), (dict(k=17), "k <= 16"),
    (dict(e=4, k=5), "k <= E"), (dict(stride=63), "stride"), (dict(groups=0), "groups"),
    (dict(groups=17), "groups"), (dict(groups=3), "groups"), (dict(groups=4, keep=0), "groups"),
    (dict(groups=4, keep=5), "groups"), (dict(groups=4, keep=2, best=3), "groups"),
    (dict(e=16, groups=8, keep=1, k=3, stride=16), "kept groups"),
])
def test_route_refusals(kw, text):
    assert text in refused("nsosx_moe_route_scored", *route(**kw))


def test_route_overflow():
    assert "too large" in refused("nsosx_moe_route_scored", *route(rows=2**31 - 1, k=2), status=2)


def test_route_rows_of_a_launch():
    """16 threads a row and fewer than 2^32 a launch."""
    assert "too large" in refused("nsosx_moe_route_scored",
                                  *route(rows=2**28, e=1, stride=1, k=1), status=2)
    assert "too large" in refused("nsosx_moe_route_scored_backward", P, 0, 1, P, P, 2**28, 1, 1, 0, 1, 1.0,
                                  P, None, status=2)


@pytest.mark.parametrize("logits,selected,dweights", [(4, 0, 1024), (1024, 4, 2048), (1024, 2048, 124)])
def test_route_backward_overlaps(logits, selected, dweights):
    """dlogits: 4 rows of 8 floats at 4 P; the input named by the small distance meets it."""
    at = 4 * P
    assert "overlaps" in refused("nsosx_moe_route_scored_backward", at + logits, 0, 8, at - 8 + selected if selected
                                 else at + 4096, at + dweights, 4, 8, 2, 0, 1, 1.0, at, None)


def test_dims_past_an_int():
    assert "too large" in refused("nsosx_moe_combine_topk", P, 0, P, P, 1, 1, 1, 2**30 + 8, 2**40, 0, None,
                                  status=2)
    assert "too large" in refused("nsosx_moe_combine_topk_backward", P, 0, 2**41, 0, P, P, None, 1, 1, 1,
                                  2**30 + 8, 2**40, P, None, status=2)
    assert "too large" in refused("nsosx_int8_gemm", P, P, P, P, None, 1, 16, 2**31 - 130, P, 0, None, status=2)
    assert "too large" in refused("nsosx_int8_gemm", P, P, P, P, None, 2**31 - 130, 16, 1, P, 0, None, status=2)
    assert "too large" in refused("nsosx_grouped_int8_gemm", P, P, 4, P, P, None, P, P, 2**30 + 1, 1, 16, 16, 0,
                                  P, 0, None, status=2)


def test_int8_overlaps():
    """y [4, 16] f32 over the codes' or the weights' last bytes, and right behind them."""
    far = 64 * P
    assert "overlaps" in refused("nsosx_int8_gemm", P, P, far, P, None, 4, 32, 16, P + 127, 0, None)
    assert "overlaps" in refused("nsosx_int8_gemm", P, P, far, P, None, 4, 32, 16, far - 255, 0, None)
    assert "overlaps" in refused("nsosx_grouped_int8_gemm", P, P, 4, far, P, None, P, None, 4, 2, 32, 16, 0,
                                 far + 1023, 0, None)
    assert "overlaps" in refused("nsosx_grouped_int8_gemm", P, P, 4, far, P, None, P, None, 4, 2, 32, 16, 0,
                                 P + 127, 0, None)


def test_route_workspace():
    lib = _lib.lib()
    assert lib.nsosx_moe_route_scored_workspace(0, 8) == 0
    assert lib.nsosx_moe_route_scored_workspace(8, 513) == 0
    assert lib.nsosx_moe_route_scored_workspace(1, 8) == 8
    for rows in (1, 65, 5000, 100000):
        assert lib.nsosx_moe_route_scored_workspace(rows, 256) >= 256 * ((rows + 63) // 64)


@pytest.mark.parametrize("args,text", [
    ((None, 0, 8, P, P, 1, 8, 2, 0, 1, 1.0, P, None), "null"),
    ((P, 3, 8, P, P, 1, 8, 2, 0, 1, 1.0, P, None), "dtype"),
    ((P, 0, 7, P, P, 1, 8, 2, 0, 1, 1.0, P, None), "stride"),
    ((P, 0, 8, P, P, 1, 8, 9, 0, 1, 1.0, P, None), "k <= E"),
    ((P, 0, 8, P, P, 0, 8, 2, 0, 1, 1.0, P, None), "rows"),
])
def test_route_backward_refusals(args, text):
    assert text in refused("nsosx_moe_route_scored_backward", *args)


@pytest.mark.parametrize("args,text", [
    ((None, 0, P, P, 4, 8, 2, 16, 2 * P, 0, None), "null"),
    ((P, 2, P, P, 4, 8, 2, 16, 2 * P, 0, None), "dtype"),
    ((P, 0, P, P, 4, 8, 17, 16, 2 * P, 0, None), "k <= 16"),
    ((P, 0, P, P, 4, 0, 2, 16, 2 * P, 0, None), "positive"),
    ((P, 0, P, P, 4, 8, 2, 16, P + 64, 0, None), "overlaps"),
])
def test_combine_refusals(args, text):
    assert text in refused("nsosx_moe_combine_topk", *args)


@pytest.mark.parametrize("args,text", [
    ((P, 0, None, 0, P, P, None, 4, 8, 2, 16, 2 * P, P, None), "null"),
    ((P, 0, P, 5, P, P, None, 4, 8, 2, 16, 2 * P, P, None), "dtype"),
    ((P, 0, P, 0, P, P, None, 4, 8, 0, 16, 2 * P, P, None), "k <= 16"),
    ((P, 0, 4 * P, 0, P, P, None, 4, 8, 2, 16, P, P, None), "overlaps"),
    ((4 * P, 0, P, 0, P, P, None, 4, 8, 2, 16, P, P, None), "overlaps"),
])
def test_combine_backward_refusals(args, text):
    assert text in refused("nsosx_moe_combine_topk_backward", *args)


@pytest.mark.parametrize("args,text,status", [
    ((None, P, P, P, None, 1, 16, 16, P, 0, None), "null", 1),
    ((P, P, P, None, None, 1, 16, 16, P, 0, None), "null", 1),
    ((P, P, P, P, None, 0, 16, 16, P, 0, None), "positive", 1),
    ((P, P, P, P, None, 1, 0, 16, P, 0, None), "positive", 1),
    ((P, P, P, P, None, 1, 16, 16, P, 2, None), "dtype", 1),
    ((P, P, P, P, None, 1, 131072, 16, P, 0, None), "131071", 2),
    ((P, P, P, P, None, 2**31 - 1, 16, 2**31 - 1, P, 0, None), "too large", 2),
])
def test_int8_refusals(args, text, status):
    assert text in refused("nsosx_int8_gemm", *args, status=status)


@pytest.mark.parametrize("args,text,status", [
    ((P, P, 4, None, P, None, P, None, 4, 2, 16, 16, 0, P, 0, None), "null", 1),
    ((P, P, 4, P, P, None, None, None, 4, 2, 16, 16, 0, P, 0, None), "null", 1),
    ((P, P, 4, P, P, None, P, None, 4, 0, 16, 16, 0, P, 0, None), "positive", 1),
    ((P, P, 4, P, P, None, P, None, 4, 1025, 16, 16, 0, P, 0, None), "1024", 1),
    ((P, P, 3, P, P, None, P, None, 4, 2, 16, 16, 0, P, 0, None), "every slot", 1),
    ((P, P, 4, P, P, None, P, None, 4, 2, 16, 16, 0, P, 7, None), "dtype", 1),
    ((P, P, 4, P, P, None, P, None, 4, 2, 200000, 16, 0, P, 0, None), "131071", 2),
    ((P, P, 4, P, P, None, P, P, 2**31 - 1, 2, 16, 2**31 - 1, 0, P, 0, None), "too large", 2),
])
def test_grouped_int8_refusals(args, text, status):
    assert text in refused("nsosx_grouped_int8_gemm", *args, status=status)


I8, F, I32 = torch.int8, torch.float32, torch.int32


@pytest.mark.parametrize("fn,text", [
    (lambda: ops.moe_route_scored(torch.zeros(4, 8), 2), "device tensor"),
    (lambda: ops.moe_route_scored_backward(torch.zeros(4, 8), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2)),
     "device tensor"),
    (lambda: ops.moe_combine_topk(torch.zeros(8, 4), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2)),
     "device tensor"),
    (lambda: ops.moe_combine_topk(torch.zeros(8), torch.zeros(4, 2, dtype=I32), torch.zeros(4, 2)),
     "expert_out"),
    (lambda: ops.int8_gemm(torch.zeros(4, 8, dtype=I8), torch.zeros(4), torch.zeros(3, 8, dtype=I8),
                           torch.zeros(3)), "device tensor"),
    (lambda: ops.int8_gemm(torch.zeros(4, 8, dtype=I8), torch.zeros(4), torch.zeros(3, 9, dtype=I8),
                           torch.zeros(3)), "agree in K"),
    (lambda: ops.grouped_int8_gemm(torch.zeros(4, 8, dtype=I8), torch.zeros(4),
                                   torch.zeros(2, 3, 9, dtype=I8), torch.zeros(2, 3),
                                   torch.zeros(3, dtype=I32)), "agree in K"),
    (lambda: ops.grouped_int8_gemm(torch.zeros(0, 8, dtype=I8), torch.zeros(0),
                                   torch.zeros(2, 3, 8, dtype=I8), torch.zeros(2, 3),
                                   torch.zeros(3, dtype=I32)), "agree in K"),
])
def test_wrapper_refusals_on_cpu_tensors(fn, text):
    with pytest.raises(ValueError, match=text):
        fn()


@pytest.mark.parametrize("meets", ["slot_of", "weights", "perm", "dweights"])
@pytest.mark.parametrize("end", ["first", "last"])
def test_combine_backward_overlaps(meets, end):
    """dexpert: 8 slots of 16 floats at 4 P, over the first or the last bytes of the small arrays (4 rows
    of k 2, 32 bytes, and 8 slots' perm, 32 too)."""
    at, far = 4 * P, {n: (8 + i) * P for i, n in enumerate(("slot_of", "weights", "perm", "dweights"))}
    far[meets] = at + 8 * 16 * 4 - 4 if end == "first" else at - 28
    text = refused("nsosx_moe_combine_topk_backward", P, 0, 2 * P, 0, far["slot_of"], far["weights"], far["perm"], 4,
                   8, 2, 16, at, far["dweights"], None)
    assert "overlaps dweights" in text if meets == "dweights" else "overlaps an input" in text
