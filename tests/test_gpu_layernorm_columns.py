"""Layer norm's gradients of rows so wide that their columns' sums are more than a launch's threads, and of
widths around the ones where a workgroup takes more columns than sixteen."""
import pytest
import torch

from reimagined_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim", [(1, 2**26 + 17), (3, 2**20 - 1), (2, 2**20 + 1), (2, 2**21 + 33)])
def test_wide(dev, rows, dim):
    torch.manual_seed(2)
    x, dy = (torch.randn((rows, dim), device=dev, dtype=torch.bfloat16) for _ in range(2))
    mean, rstd = torch.full((rows,), 0.25, device=dev), torch.full((rows,), 1.5, device=dev)
    g = ops.layernorm_backward(dy, x, mean, rstd)
    # one to three rows: each term is (x - mean) rstd dy with a rounding each, then an add each
    term = (x.double() - 0.25) * 1.5 * dy.double()
    lim = (4 + rows) * 2.0**-24 * term.abs().sum(0)
    assert ((g["dweight"].double() - term.sum(0)).abs() <= lim).all()
    lim = (1 + rows) * 2.0**-24 * dy.double().abs().sum(0)
    assert ((g["dbias"].double() - dy.double().sum(0)).abs() <= lim).all()
    assert torch.isfinite(g["dx"]).all()
