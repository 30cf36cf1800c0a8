"""Layer norm, the gated recurrence, its step and the balance loss where elements lie past 2^31 of their
tensors: what is computed there against small calls of the same rows or channels, bit for bit."""
import pytest
import torch

from reimagined_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rand(dev, rows, cols, dtype, seed):
    """rows x cols without a random number for each: a block of rows again and again."""
    g = torch.Generator(device=dev).manual_seed(seed)
    part = torch.randn((4099, cols), generator=g, device=dev, dtype=F32).to(dtype)
    out = torch.empty((rows, cols), dtype=dtype, device=dev)
    for r in range(0, rows, 4099):
        out[r:r + 4099] = part[:min(4099, rows - r)]
    return out


def test_layernorm(dev):
    rows, dim = 2**21 + 5, 1030
    x = rand(dev, rows, dim, BF16, 1)
    w = torch.linspace(0.5, 1.5, dim, device=dev)
    res, y, mean, rstd = ops.add_layernorm(x, x, w, w, want_stats=True)
    cut = slice(rows - 70, rows)
    sres, sy, smean, srstd = ops.add_layernorm(x[cut], x[cut], w, w, want_stats=True)
    assert torch.equal(res[cut], sres) and torch.equal(y[cut], sy)
    assert torch.equal(mean[cut], smean) and torch.equal(rstd[cut], srstd)
    g = ops.layernorm_backward(y, res, mean, rstd, w, dresidual=x)
    s = ops.layernorm_backward(sy, sres, smean, srstd, w, dresidual=x[cut])
    assert torch.equal(g["dx"][cut], s["dx"])
    assert torch.isfinite(g["dweight"]).all() and torch.isfinite(g["dbias"]).all()


def test_recurrence(dev):
    t, d = 2**20 + 77, 2050
    x, rg, ig = (rand(dev, t, d, BF16, s) for s in (2, 3, 4))
    lam = torch.linspace(-6.0, -3.0, d, device=dev)
    cu = torch.tensor([0, 1000, t - 300, t - 1], dtype=torch.int32, device=dev)
    y, final, carry = ops.gated_recurrence(x, rg, ig, lam, cu, want_carry=True)
    lo = d - 70
    p = [v[:, lo:].contiguous() for v in (x, rg, ig)]
    sy, sfinal, scarry = ops.gated_recurrence(*p, lam[lo:].contiguous(), cu, want_carry=True)
    assert torch.equal(y[:, lo:], sy) and torch.equal(final[:, lo:], sfinal) and torch.equal(carry[:, lo:], scarry)
    assert not y[t - 1:].any()
    g = ops.gated_recurrence_backward(y, x, rg, ig, lam, cu, carry)
    s = ops.gated_recurrence_backward(sy, *p, lam[lo:].contiguous(), cu, scarry)
    for k in s:
        assert torch.equal(g[k][..., lo:], s[k]), k


def test_step(dev):
    rows, d = 262140, 8200
    x = rand(dev, rows, d, BF16, 5)
    lam = torch.linspace(-6.0, -3.0, d, device=dev)
    state = torch.full((rows, d), 0.25, device=dev)
    cut = slice(rows - 9, rows)
    small = state[cut].clone()
    y = ops.gated_recurrence_step(x, x, x, lam, state)
    sy = ops.gated_recurrence_step(x[cut], x[cut], x[cut], lam, small)
    assert torch.equal(y[cut], sy) and torch.equal(state[cut], small)
    with pytest.raises(ops.NsosxError, match="too large"):
        ops.gated_recurrence_step(*(torch.zeros((262141, 1), device=dev) for _ in range(3)), lam[:1].contiguous(),
                                  torch.zeros((262141, 1), device=dev))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance(dev, score):
    rows, e, k = 1024 * 4099, 512, 2
    logits = rand(dev, rows, e, F32, 6)
    sel = torch.stack([torch.arange(rows, device=dev) % e, torch.arange(rows, device=dev) % 7 + 300], 1).int()
    f = ops.moe_balance_loss(logits, sel, score=score)
    assert torch.equal(f["counts"][0].long(), torch.bincount(sel.view(-1), minlength=e))
    assert f["tokens"].tolist() == [rows]
    # 4099 rows again and again: their mean.  64 rows a block and 16 runs of blocks, added one after the other:
    # 4099 adds and some forty, each off by half a step at most; the small call is off by less than a hundred.
    want = ops.moe_balance_loss(logits[:4099], sel[:4099], score=score)["mean_prob"]
    assert ((f["mean_prob"] - want).abs() <= 4300 * 2.0**-24 * want).all()
    cut = slice(rows - 40, rows)
    d = ops.moe_balance_loss_backward(logits, f["counts"], f["tokens"], k, score=score)
    s = ops.moe_balance_loss_backward(logits[cut], f["counts"], f["tokens"], k, score=score)
    assert torch.equal(d[cut], s)
