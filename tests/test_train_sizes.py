"""Sizes that an int of the C entries cannot hold are refused, not cut to their lowest 32 bits (CPU only, on
tensors of one element seen as many)."""
import pytest
import torch

from reimagined_amd import ops

MANY = 2**32 + 5


def wide(*shape, dtype=torch.float32):
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(*shape)


@pytest.mark.parametrize("shape", [(MANY, 8), (8, MANY), (2**31, 8)])
def test_layernorm(shape):
    x, row = wide(*shape), wide(shape[0])
    for f in (lambda: ops.layernorm(x), lambda: ops.add_layernorm(x, x),
              lambda: ops.layernorm_backward(x, x, row, row)):
        with pytest.raises(ValueError, match="less than 2\\^31"):
            f()


@pytest.mark.parametrize("shape", [(MANY, 8), (8, MANY), (2**31, 8)])
def test_recurrence(shape):
    x, lam, cu = wide(*shape), wide(shape[1]), torch.tensor([0, 4], dtype=torch.int32)
    for f in (lambda: ops.gated_recurrence(x, x, x, lam, cu), lambda: ops.gated_recurrence_step(x, x, x, lam, x),
              lambda: ops.gated_recurrence_backward(x, x, x, x, lam, cu, x)):
        with pytest.raises(ValueError, match="less than 2\\^31"):
            f()


def test_sequences():
    x, lam, cu = torch.zeros(4, 8), torch.zeros(8), wide(MANY, dtype=torch.int32)
    with pytest.raises(ValueError, match="less than 2\\^31"):
        ops.gated_recurrence(x, x, x, lam, cu)
    with pytest.raises(ValueError, match="less than 2\\^31"):
        ops.gated_recurrence_backward(x, x, x, x, lam, cu, x)


def test_logits():
    x, sel, counts = wide(MANY, 8), wide(MANY, 2, dtype=torch.int32), torch.zeros((1, 8), dtype=torch.int32)
    for f in (lambda: ops.moe_balance_loss(x, sel), lambda: ops.moe_balance_loss_backward(x, counts, counts[0, :1], 2),
              lambda: ops.moe_route_scored(x, 2)):
        with pytest.raises(ValueError, match="less than 2\\^31"):
            f()
