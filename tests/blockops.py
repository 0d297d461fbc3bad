"""The gated block's operators in 64 bits, run through their layers, and the error that a kernel may have (test helper).

Tolerances follow from the arithmetic, to first order in the unit u of fp32 (2^-24): a sum of n terms in any order is off by at most
n u sum |terms|, a product or a difference by u of it, an output besides by half a step of its type.  A tenth is added for the
second order."""
import numpy as np

from tests import headops as ho

U = ho.U32
KINDS = ["none", "rms", "layer"]


def out_error(exact, err, dtype):
    err = 1.1 * err
    return err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype]


class Norm:
    """A norm's rows in 64 bits, and errors of the kernel's fp32 statistics and normed values for inputs that are off by `err`."""

    def __init__(self, x, kind, eps, err=0.0):
        n = x.shape[1]
        err = np.broadcast_to(err, x.shape)
        mean = x.mean(1, keepdims=True) if kind == "layer" else np.zeros((len(x), 1))
        self.kind = kind
        if kind == "none":
            self.mean, self.rstd, self.hat, self.hat_err = mean[:, 0], np.ones(len(x)), x, err
            return
        d = x - mean
        rstd = 1 / np.sqrt((d ** 2).mean(1, keepdims=True) + eps)
        hat = d * rstd
        mean_err = (n * U * np.abs(x).mean(1, keepdims=True) + err.mean(1, keepdims=True) + U * np.abs(mean)) * (kind == "layer")
        d_err = err + mean_err + U * np.abs(d)
        # 1 / sqrt(v + eps): half the relative error of v + eps, which is of positive terms, and a handful of roundings
        rel = rstd[:, 0:1] ** 2 * (np.abs(d) * d_err).mean(1, keepdims=True) + (0.5 * n + 6) * U
        self.mean, self.rstd, self.hat = mean[:, 0], rstd[:, 0], hat
        self.mean_err, self.rstd_err = 1.1 * mean_err[:, 0], 1.1 * (rel * rstd)[:, 0]
        self.hat_err = d_err * rstd + np.abs(hat) * (rel + U)


def norms(x, block, gate, ag, ab, bg, bb, after, before, scale, eps):
    """stream, its error, output, its error, the two norms; every parameter an array (ones and zeros where there is none)"""
    first = None
    stream, err = x, 0.0
    if block is not None:
        first = Norm(block, after, eps)
        P, Q = scale * gate * ag, scale * gate * ab
        stream = x + first.hat * P + Q
        err = np.abs(P) * first.hat_err + U * (5 * np.abs(first.hat * P) + 4 * np.abs(Q) + 2 * np.abs(x))
    second = Norm(stream, before, eps, err)
    y = second.hat * bg + bb
    yerr = np.abs(bg) * second.hat_err + U * (3 * np.abs(second.hat * bg) + np.abs(bb))
    return stream, err, y, yerr, first, second


def _through(g, gerr, hat, hat_err, rstd, kind):
    """rstd (g - mean g - hat mean (g hat)) and its error"""
    if kind == "none":
        return g, gerr
    n = g.shape[1]
    gm = g.mean(1, keepdims=True) * (kind == "layer")
    gm_err = (gerr.mean(1, keepdims=True) + (n + 1) * U * np.abs(g).mean(1, keepdims=True)) * (kind == "layer")
    p = (g * hat).mean(1, keepdims=True)
    p_err = (gerr * np.abs(hat) + np.abs(g) * hat_err).mean(1, keepdims=True) + (n + 3) * U * np.abs(g * hat).mean(1, keepdims=True)
    v = g - gm - hat * p
    err = gerr + gm_err + np.abs(hat) * p_err + hat_err * np.abs(p) + 3 * U * (np.abs(g) + np.abs(gm) + np.abs(hat * p))
    r = rstd[:, None]
    return v * r, err * r + 2 * U * np.abs(v * r)


def _hat(x, mean, rstd, kind):
    """Normed values of given fp32 statistics, and the error of making them in fp32."""
    if kind == "none":
        return x, np.zeros_like(x)
    mean = mean[:, None] if kind == "layer" else 0.0
    hat = (x - mean) * rstd[:, None]
    return hat, 3 * U * (np.abs(x) + np.abs(mean)) * rstd[:, None]


def norms_grad(stream, block, gate, ag, ab, bg, stats, dy, ds, after, before, scale):
    """{name: (gradient, error)} of the stream, the block and the parameters"""
    m = len(stream)
    zero = np.zeros_like(stream)
    d, derr = (zero if ds is None else ds), zero
    out = {}
    if dy is not None:
        xh, xerr = _hat(stream, stats.get("before_mean"), stats.get("before_rstd"), before)
        t, terr = _through(dy * bg, U * np.abs(dy * bg), xh, xerr, stats.get("before_rstd"), before)
        derr = terr + 2 * U * (np.abs(d) + np.abs(t))
        d = d + t
        out["before_gamma"] = (dy * xh).sum(0), (np.abs(dy) * xerr + (m + 2) * U * np.abs(dy * xh)).sum(0)
        out["before_beta"] = dy.sum(0), m * U * np.abs(dy).sum(0)
    out["stream"] = d, derr
    if block is None:
        return out
    P = scale * gate * ag
    yh, yerr = _hat(block, stats.get("after_mean"), stats.get("after_rstd"), after)
    h, herr = d * P, np.abs(P) * derr + 4 * U * np.abs(d * P)
    out["block"] = _through(h, herr, yh, yerr, stats.get("after_rstd"), after)
    A, Aerr = (d * yh).sum(0), (derr * np.abs(yh) + np.abs(d) * yerr + (m + 2) * U * np.abs(d * yh)).sum(0)
    B, Berr = d.sum(0), (derr + m * U * np.abs(d)).sum(0)
    out["gate"] = scale * (ag * A + ab * B), np.abs(scale) * (np.abs(ag) * Aerr + np.abs(ab) * Berr + 5 * U * (np.abs(ag * A) + np.abs(ab * B)))
    out["after_gamma"] = scale * gate * A, np.abs(scale * gate) * (Aerr + 4 * U * np.abs(A))
    out["after_beta"] = scale * gate * B, np.abs(scale * gate) * (Berr + 4 * U * np.abs(B))
    return out


def loss(x, w, b, t, g=None):
    """Loss, logsumexp and (g given) {name: (gradient, its error)}, with the errors of the first two, of fp32 logits; rows of finite logits, or
    whose bias forbids classes (-inf)."""
    k, n = x.shape[1], len(w)
    bias = 0.0 if b is None else b
    z = x @ w.T + bias
    shared = np.where(np.isfinite(bias), np.abs(bias), 0.0)
    zerr = (k + 1) * U * (np.abs(x) @ np.abs(w).T + shared)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = z.max(1)
        safe = np.where(m == -np.inf, 0.0, m)
        e = np.exp(z - safe[:, None])
        lse = safe + np.log(e.sum(1))
        p = np.exp(z - np.where(lse == -np.inf, 0.0, lse)[:, None])
        given = (t >= 0) & (t < n)
        at = np.where(given, t, 0)
        zt, rows = z[np.arange(len(x)), at], np.arange(len(x))
        out = np.where(t < 0, 0.0, np.where(t >= n, np.nan, np.where(zt == -np.inf, np.inf, lse - zt)))
    # exp's argument is off by its rounding and by the logits' error, exp by some units, the sum by one a term; the logarithm by that relative error
    far = np.where(np.isfinite(z), np.abs(z - safe[:, None]), 0.0)
    rel = zerr + U * (4 * far + 6)
    serr = (p * rel).sum(1) + (n + 8) * U
    lse_err = 1.1 * (serr + 4 * U * (np.abs(np.where(np.isfinite(lse), lse, 0)) + np.abs(np.log(n + 1.0))))
    loss_err = lse_err + zerr[rows, at] + 4 * U * (np.abs(safe - np.where(np.isfinite(zt), zt, safe)) + np.log(n + 1.0))
    if g is None:
        return out, loss_err, lse, lse_err
    return out, loss_err, lse, lse_err, z, zerr, p


def loss_grads(x, w, t, g, z, zerr, p, lse, lse_err, dtype):
    """{name: (gradient, error)}: d as the products read it is off by its own rounding and by what its logits and logsumexp are off by"""
    m, k = x.shape
    n = len(w)
    none = (t < 0) | (lse == -np.inf)
    g = np.where(none, 0.0, g)
    one = np.zeros((m, n))
    one[np.arange(m), np.where(t < 0, 0, t)] = 1.0
    d = g[:, None] * (p - one)
    zabs = np.where(np.isfinite(z), np.abs(z), 0.0)
    derr = np.abs(g)[:, None] * (p * (zerr + lse_err[:, None] + U * (4 * zabs + 4 * np.abs(np.where(np.isfinite(lse), lse, 0))[:, None] + 6)) + U * np.abs(p - one)) * 1.1
    # f16: d is scaled, so that what lies below the normal numbers is less than 2^-38 of the largest |g|
    tiny = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -38 * np.abs(g).max()}[dtype]
    # (of 256 rows at most d is kept in two planes: its rounding, and what that left, rounded)
    step = ho.U[dtype] ** 2 if dtype != "f32" and m <= 256 else ho.U[dtype]
    used = derr + step * (np.abs(d) + derr) + tiny
    out = {}
    terms, exact = np.abs(d) @ np.abs(w), d @ w
    out["input"] = exact, used @ np.abs(w) + (n + 32) * U * 1.01 * terms
    terms, exact = np.abs(d).T @ np.abs(x), d.T @ x
    out["weight"] = exact, used.T @ np.abs(x) + m * U * 1.01 * terms
    out["bias"] = d.sum(0), derr.sum(0) + m * U * 1.01 * np.abs(d).sum(0)
    return out
