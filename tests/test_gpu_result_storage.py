"""What layer norm, the gated recurrence and the balance loss return holds the results alone, no workspace."""
import pytest
import torch

from reimagined_amd import ops

pytestmark = pytest.mark.gpu


def held(results):
    """Bytes of the storages behind some tensors, and of the tensors themselves."""
    results = [t for t in results if t is not None]
    storages = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in results}
    return sum(storages.values()), sum(t.numel() * t.element_size() for t in results)


@pytest.mark.parametrize("rows,dim", [(1, 5), (4096, 64), (2048, 2048), (300, 17000)])
def test_layernorm(dev, rows, dim):
    x = torch.randn((rows, dim), device=dev)
    y, mean, rstd = ops.layernorm(x, want_stats=True)
    assert held([y, mean, rstd])[0] == held([y, mean, rstd])[1]
    g = ops.layernorm_backward(x, x, mean, rstd)
    assert held(g.values())[0] == held(g.values())[1]
    assert all(held([t])[0] == held([t])[1] for t in g.values())


@pytest.mark.parametrize("rows,e,lens", [(1, 8, None), (4096, 256, None), (1000, 60, [400, 0, 600])])
def test_balance(dev, rows, e, lens):
    logits = torch.randn((rows, e), device=dev)
    sel = torch.zeros((rows, 2), dtype=torch.int32, device=dev)
    sel[:, 1] = 1
    cu = None if lens is None else torch.tensor([0, 400, 400, 1000], dtype=torch.int32, device=dev)
    f = ops.moe_balance_loss(logits, sel, cu_seqlens=cu)
    assert all(held([t])[0] == held([t])[1] for t in f.values())


def test_recurrence(dev):
    x, lam = torch.randn((999, 70), device=dev), torch.zeros(70, device=dev)
    cu = torch.tensor([0, 500, 999], dtype=torch.int32, device=dev)
    out = ops.gated_recurrence(x, x, x, lam, cu, want_carry=True)
    assert held(out)[0] == held(out)[1]
    g = ops.gated_recurrence_backward(x, x, x, x, lam, cu, out[2])
    assert held(g.values())[0] == held(g.values())[1]
