"""The float64 definitions that the training operators are tested against, against differences of
their own forward (CPU only)."""
import numpy as np
import pytest

import train_ref as ref


def differences(f, args, grads, rng, step=1e-6, tol=1e-6):
    """Directional derivatives of f by central differences against the gradients' products."""
    for name, g in grads.items():
        v = rng.standard_normal(args[name].shape)
        hi, lo = (f(**{**args, name: args[name] + s * step * v}) for s in (1, -1))
        want = (hi - lo) / (2 * step)
        assert abs(want - (g * v).sum()) <= tol * max(1.0, abs(want), np.abs(g * v).sum()), name


def test_layernorm_gradient():
    rng = np.random.default_rng(1)
    x, w, b = rng.standard_normal((5, 13)) + 0.4, rng.standard_normal(13), rng.standard_normal(13)
    dy = rng.standard_normal((5, 13))

    def f(x, w, b):
        return float((ref.layernorm(x, w, b, 1e-5)[0] * dy).sum())

    _, mean, rstd, *_ = ref.layernorm(x, w, b, 1e-5)
    dx, _, dw, _, db, _ = ref.layernorm_backward(dy, x, mean, rstd, w, None)
    differences(f, dict(x=x, w=w, b=b), dict(x=dx, w=dw, b=db), rng)


def test_recurrence_gradient():
    rng = np.random.default_rng(2)
    t, d, cu = 23, 5, [0, 4, 4, 17, 23]
    args = dict(x=rng.standard_normal((t, d)), rg=rng.standard_normal((t, d)),
                ig=rng.standard_normal((t, d)), lam=rng.normal(-4, 1, d), h0=rng.standard_normal((4, d)))
    dy, dfinal = rng.standard_normal((t, d)), rng.standard_normal((4, d))

    def f(x, rg, ig, lam, h0):
        r = ref.Recurrence(x, rg, ig, lam, cu, 8.0, h0)
        return float((r.h * dy).sum() + (r.final * dfinal).sum())

    g = ref.Recurrence(cu=cu, rate=8.0, **args).backward(dy, dfinal)
    differences(f, args, dict(x=g["dx"][0], rg=g["drg"][0], ig=g["dig"][0], lam=g["dlam"][0],
                              h0=g["dinitial"][0]), rng)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance_gradient(score):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((12, 7))
    sel = np.argsort(-x, axis=1)[:, :3]
    valid = rng.random(12) < 0.8
    cu = [0, 5, 5, 12]

    def f(x):
        return float(ref.balance(x, sel, score, cu, valid, 1.0)[0])

    differences(f, dict(x=x), dict(x=ref.balance(x, sel, score, cu, valid, 1.0)[4]), rng)
