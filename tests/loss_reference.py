"""The choice losses in 64 bits, from their formulas, with the error bounds that
32-bit kernels are held to."""
import math

import numpy as np

EPS = 2.0 ** -24  # unit roundoff of fp32
ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -133}  # half a subnormal step, or one


def softmax_rows(z, label):
    """(log p of the label, top, log sum, p) of margins [R, K] in 64 bits; rows
    without a label give zeros, rows without a class -inf."""
    rows, classes = z.shape
    live = (label >= 0) & (label < classes)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top = z.max(1) if classes else np.zeros(rows)
        none = live & (top == -np.inf)
        base = np.where(none, 0.0, top)
        e = np.exp(z - base[:, None])
        s = e.sum(1)
        log_sum = np.where(none, 0.0, np.log(s))
        p = np.where(none[:, None], 0.0, e / s[:, None])
        chosen = z[np.arange(rows), np.where(live, label, 0)] if rows else np.zeros(0)
        logp = np.where(none, -np.inf, (chosen - base) - log_sum)
    zero = lambda v: np.where(live, v, 0.0)  # noqa: E731
    return zero(logp), zero(top), zero(log_sum), p, live, none


def log_prob_bound(z, label, logp, top, log_sum):
    """Bound on |log p - its fp32 value|: every exponential is off by a few
    roundings of itself and of its argument (whose weighted mean is at most
    log K), a sum of K terms in chains of at most 512 by 512 EPS, the logarithm
    and the two subtractions by one rounding each."""
    classes = z.shape[1]
    rel = EPS * (520 + 4 * math.log(classes + 1))
    with np.errstate(invalid="ignore"):
        gap = np.abs(np.where(np.isfinite(logp), logp + log_sum, 0.0))
    return rel + 4 * EPS * (np.abs(log_sum) + gap + 1)


def grad_rows(z, label, p, c, live, none):
    """Gradient and curvature of sum c * log p(label)."""
    rows, classes = z.shape
    c = np.where(live & ~none, c, 0.0)
    hit = np.zeros((rows, classes))
    if rows:
        hit[np.arange(rows), np.where(live, label, 0)] = 1.0
    zero = (c == 0.0)[:, None]
    with np.errstate(invalid="ignore"):
        g = np.where(zero, 0.0, c[:, None] * (hit - p))
        h = np.where(zero, 0.0, np.abs(c)[:, None] * np.maximum(2 * p * (1 - p), 1e-16))
    return g, h


def grad_bound(z, top, p, c, c_err, g, h, dtype):
    """Bounds of the gradient and the curvature: p is off by the sum's and the
    exponential's relative error, c by c_err; a gradient is rounded to its type."""
    classes = z.shape[1]
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.where(np.isfinite(z), np.minimum(np.abs(z - top[:, None]), 200.0), 200.0)
    rel = EPS * (530 + 4 * math.log(classes + 1) + 8 * x)
    ac, ce = np.abs(c)[:, None], np.broadcast_to(np.asarray(c_err, np.float64), c.shape)[:, None]
    dg = (ac + ce) * p * rel + ce + 4 * EPS * ac + 4 * EPS * np.abs(g)
    dg = dg + ROUND[dtype] * (np.abs(g) + dg) * 1.01 + TINY[dtype]
    dh = 2 * ((ac + ce) * 2 * p * rel + ce * (p + 1e-16) + 8 * EPS * np.abs(h)) + 2 * EPS * ac + 1e-38
    return dg, dh


def policy(logp, old, adv, ref, weight, clip, kl):
    """(loss, derivative by log p, |its| parts for a bound, distance of the ratio from the nearer clip edge)."""
    with np.errstate(over="ignore", invalid="ignore"):
        w = np.ones_like(logp) if weight is None else weight
        r = np.exp(logp - old)
        s1, s2 = r * adv, np.clip(r, 1 - clip[0], 1 + clip[1]) * adv
        loss, c = -np.minimum(s1, s2), np.where(s1 <= s2, -s1, 0.0)
        size = np.abs(s1)
        if ref is not None:
            d = ref - logp
            loss = loss + kl * (np.expm1(d) - d)
            c = c - kl * np.expm1(d)
            size = size + kl * (np.exp(d) + np.abs(d) + 1)
        zero = w == 0
        edge = np.minimum(np.abs(r - (1 - clip[0])), np.abs(r - (1 + clip[1])))
    return np.where(zero, 0.0, w * loss), np.where(zero, 0.0, w * c), np.abs(w) * size, edge, r


def pair_terms(x, smoothing):
    """(loss, derivative, second derivative) by x."""
    a = np.abs(x)
    e = np.exp(-a)
    small = np.log1p(e)
    up, down = np.where(x >= 0, 1 / (1 + e), e / (1 + e)), np.where(x >= 0, e / (1 + e), 1 / (1 + e))
    loss = (1 - smoothing) * (np.maximum(-x, 0) + small) + smoothing * (np.maximum(x, 0) + small)
    return loss, smoothing * up - (1 - smoothing) * down, up * down


def item_sums(v, begin):
    run = np.concatenate([[0.0], np.cumsum(v)])
    return run[begin[1:]] - run[begin[:-1]]
