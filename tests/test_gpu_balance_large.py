"""The balance loss's mean probabilities over millions of rows, within the depth of their sums."""
import pytest
import torch

from reimagined_amd import ops

pytestmark = pytest.mark.gpu


def depth(rows):
    """Adds behind one another in a column's sum: the steps of a lane's rows (of 64, as many for each of 512 blocks
    as it takes), the block's 4 rows a wave and 16 waves, a 16th of the blocks, 16 of them, the division."""
    steps = -(-(-(-rows // 64)) // 512)
    blocks = -(-rows // (64 * steps))
    return steps + 2 + 15 + -(-blocks // 16) + 15 + 1


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("times", [3, 64, 1024])
def test_mean_of_repeated_rows(dev, score, times):
    """4099 rows again and again have the same mean: both sums are of numbers above 0, so each add is off by half a
    step of what it has at most."""
    e, part = 512, 4099
    g = torch.Generator(device=dev).manual_seed(6)
    few = torch.randn((part, e), generator=g, device=dev)
    logits = few.repeat(times, 1)
    sel = (torch.arange(part * times, device=dev, dtype=torch.int32) % e).view(-1, 1).contiguous()
    f = ops.moe_balance_loss(logits, sel, score=score)
    want = ops.moe_balance_loss(few, sel[:part].contiguous(), score=score)["mean_prob"].double()
    lim = (depth(part * times) + depth(part)) * 2.0**-24 * (1 + 2.0**-14)
    assert ((f["mean_prob"].double() - want).abs() <= lim * want).all()
