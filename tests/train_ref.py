"""Float64 definitions of layer norm, the gated recurrence and the balance loss, with bounds of what
a float32 evaluation of the same formulas may be off, each rounding counted as half a step (U)."""
import numpy as np

U = 2.0**-24
HALF_STEP = {"f32": 2.0**-24, "bf16": 2.0**-8}  # of the stored result, relative


def sig(x):
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1 / (1 + e), e / (1 + e))


def softplus(x):
    return np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))


# ---- layer norm -------------------------------------------------------------------

def layernorm(s, w, b, eps):
    """-> y, mean, rstd and the bound of a float32 y: `depth` adds in a chain or tree of a row's sum,
    a centred variance (an error of the mean enters it squared only), five more roundings."""
    dim = s.shape[1]
    mean = s.mean(1, keepdims=True)
    d = s - mean
    var = (d * d).mean(1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    n = d * rstd
    w = np.ones(dim) if w is None else w
    b = np.zeros(dim) if b is None else b
    depth = 64 + dim / 1024
    dmean = (depth + 2) * U * np.abs(s).mean(1, keepdims=True)
    # (dmean enters the variance squared: rstd by half of dmean^2 rstd^2, relative)
    lim = np.abs(w) * (np.abs(n) * ((depth / 2 + 8) * U + dmean**2 * rstd**2) + dmean * rstd)
    lim = lim + 3 * U * (np.abs(n * w) + np.abs(b))
    drel = (depth / 2 + 6) * U + dmean[:, 0]**2 * rstd[:, 0]**2
    return n * w + b, mean[:, 0], rstd[:, 0], lim, dmean[:, 0] + U * np.abs(mean[:, 0]), drel


def layernorm_backward(dy, x, mean, rstd, w, dres):
    """-> dx, dw, db with their bounds, mean and rstd taken as given."""
    rows, dim = x.shape
    q = rstd[:, None]
    n = (x - mean[:, None]) * q
    w = np.ones(dim) if w is None else w
    g = dy * w
    m1, m2 = g.mean(1, keepdims=True), (g * n).mean(1, keepdims=True)
    dx = q * (g - m1 - n * m2)
    depth = 64 + dim / 1024
    e1 = (depth + 3) * U * np.abs(g).mean(1, keepdims=True)
    e2 = (depth + 7) * U * np.abs(g * n).mean(1, keepdims=True)
    lim = q * (e1 + np.abs(n) * e2 + 6 * U * (np.abs(g) + np.abs(m1) + np.abs(n * m2)))
    if dres is not None:
        dx = dx + dres
        lim = lim + U * np.abs(dx)
    cols = 128 + rows / 64  # adds behind one another, at most
    dw, db = (dy * n).sum(0), dy.sum(0)
    return (dx, lim, dw, (cols + 4) * U * np.abs(dy * n).sum(0), db, (cols + 1) * U * np.abs(dy).sum(0))


# ---- gated recurrence --------------------------------------------------------------

class Recurrence:
    """Forward and gradients of one packed batch, token after token, with the bounds' own
    recursions: every decay off by `ea`, every input by a share `eu`."""

    def __init__(self, x, rg, ig, lam, cu, rate, h0):
        self.x, self.cu = x, [int(c) for c in cu]
        self.t, self.d = x.shape
        self.sr, self.nr, self.si, self.ni = sig(rg), sig(-rg), sig(ig), sig(-ig)
        self.lam, self.rate = lam, rate
        self.g = rate * softplus(lam) * self.sr
        self.a = np.exp(-self.g)
        self.beta = np.sqrt(-np.expm1(-2 * self.g))
        self.u = self.beta * self.si * x
        # sigmoid: 2 |x| U of the exponent, 5 U of exponential, sum and reciprocal
        self.esr, self.esi = (2 * np.abs(rg) + 5) * U, (2 * np.abs(ig) + 5) * U
        self.eg = self.esr + 8 * U
        self.ea = self.a * (self.g * self.eg + 5 * U)     # absolute; 2 U of the tiles' products in it
        self.eb = self.eg / 2 + 9 * U                     # relative, of beta
        self.eu = self.eb + self.esi + 4 * U
        s = len(self.cu) - 1
        self.h0 = np.zeros((s, self.d)) if h0 is None else h0
        self.h, self.before = np.zeros_like(x), np.zeros_like(x)
        self.eh, self.ebefore = np.zeros_like(x), np.zeros_like(x)
        self.final, self.efinal = self.h0.copy(), np.zeros((s, self.d))
        for i in range(s):
            h, e = self.h0[i], np.zeros(self.d)
            for t in range(self.cu[i], self.cu[i + 1]):
                self.before[t], self.ebefore[t] = h, e
                hn = self.a[t] * h + self.u[t]
                e = self.a[t] * e + np.abs(h) * self.ea[t] + np.abs(self.u[t]) * self.eu[t] + 2 * U * np.abs(hn)
                h = hn
                self.h[t], self.eh[t] = h, e
            self.final[i], self.efinal[i] = h, e
        # twice the plain recursion's bound: the tiles' pairs (A, H) round on their own way as well
        self.eh, self.ebefore, self.efinal = 2 * self.eh, 2 * self.ebefore, 2 * self.efinal

    def backward(self, dy, dfinal=None):
        a, g, beta, si, x = self.a, self.g, self.beta, self.si, self.x
        dh, edh = np.zeros_like(x), np.zeros_like(x)
        s = len(self.cu) - 1
        d0 = np.zeros((s, self.d)) if dfinal is None else dfinal.copy()
        e0 = np.zeros((s, self.d))
        for i in range(s):
            m, e = d0[i], np.zeros(self.d)
            for t in range(self.cu[i + 1] - 1, self.cu[i] - 1, -1):
                dh[t] = dy[t] + m
                edh[t] = e + U * np.abs(dh[t])
                m = a[t] * dh[t]
                e = a[t] * edh[t] + np.abs(dh[t]) * self.ea[t] + U * np.abs(m)
            d0[i], e0[i] = m, 2 * e
        edh = 2 * edh
        inside = np.zeros((self.t, 1), bool)
        inside[self.cu[0]:self.cu[-1]] = True
        bent = np.divide(g * a * a, beta, out=np.zeros_like(g), where=beta > 0)
        up, down = si * x * bent, a * g * self.before
        ev = np.where(inside, dh * (up - down), 0.0)
        rela = np.divide(self.ea, a, out=np.zeros_like(a), where=a > 0)
        eev = edh * np.abs(up - down) + np.abs(dh) * (
            np.abs(up) * (self.esi + 2 * self.eg + 2 * rela + self.eb + 10 * U)
            + np.abs(down) * (self.eg + rela + 6 * U) + a * g * self.ebefore)
        eev = np.where(inside, eev, 0.0)
        dx = np.where(inside, dh * beta * si, 0.0)
        edx = edh * beta * si + np.abs(dx) * (self.eb + self.esi + 4 * U)
        dig = dx * x * self.ni
        edig = edx * np.abs(x) * self.ni + np.abs(dig) * (self.esi + 4 * U)
        drg = ev * self.nr
        edrg = eev * self.nr + np.abs(drg) * (self.esr + 2 * U)
        c = sig(self.lam) / softplus(self.lam)
        dlam = c * ev.sum(0)
        edlam = c * (eev.sum(0) + (64 + self.t / 128) * U * np.abs(ev).sum(0)) + 10 * U * np.abs(dlam)
        return {"dx": (dx, edx), "drg": (drg, edrg), "dig": (dig, edig), "dlam": (dlam, edlam),
                "dinitial": (d0, e0)}


# ---- balance loss -------------------------------------------------------------------

def balance(x, sel, score, cu, valid, dloss):
    """-> loss, counts, tokens, mean and dx of logits x [rows, E]; the gradient's bound."""
    rows, experts = x.shape
    k = sel.shape[1]
    if score == "sigmoid":
        raw, slope = sig(x), sig(-x)
        reach = np.abs(x)
    else:
        raw, slope = np.exp(x - x.max(1, keepdims=True)), 1.0
        reach = x.max(1, keepdims=True) - x
    p = raw / raw.sum(1, keepdims=True)
    ok = np.ones(rows, bool) if valid is None else np.asarray(valid) != 0
    bounds = [0, rows] if cu is None else [int(c) for c in cu]
    s = len(bounds) - 1
    counts, tokens = np.zeros((s, experts), np.int64), np.zeros(s, np.int64)
    mean, dx, lim = np.zeros((s, experts)), np.zeros_like(x), np.zeros_like(x)
    loss, some = 0.0, 0
    for i in range(s):
        mine = np.arange(bounds[i], bounds[i + 1])
        mine = mine[ok[mine]]
        tokens[i] = len(mine)
        if not len(mine):
            continue
        some += 1
        named = sel[mine].reshape(-1)
        counts[i] = np.bincount(named[(named >= 0) & (named < experts)], minlength=experts)
        mean[i] = p[mine].mean(0)
        f = experts / (k * len(mine))
        loss += f * float(counts[i] @ mean[i])
        dot = p[mine] @ counts[i]
        f = dloss * f / len(mine)
        dx[mine] = f * p[mine] * (counts[i] - dot[:, None])
        # the exponent's 2 U a unit, the row's sums of up to 64 adds, twelve single roundings
        ep = (2 * np.where(p[mine] > 0, reach[mine], 0.0) + 80) * U
        lim[mine] = f * p[mine] * (counts[i] + dot[:, None]) * (2 * ep.max(1, keepdims=True) + 12 * U)
    some = max(some, 1)
    if score == "sigmoid":
        dx, lim = dx * slope, lim * slope
    return loss / some, counts, tokens, mean, dx / some, lim / some
