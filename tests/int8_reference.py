"""Plain 64-bit restatements of the 8-bit integer operators and the expert router, on the CPU, with bounds of what float32
steps and one rounding of the result may add: what their tests compare with."""
import numpy as np
import torch

EPS = 2.0 ** -24  # half a step of float32


def quantize(x):
    """x [rows, K] -> (codes int64, scales float32 as float64). Quotients of float32 numbers, rounded exactly: their
    distance to a border is at least 2^-33 of them, which float64 tells apart."""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(1)
    bad = ~np.isfinite(x).all(1)
    with np.errstate(invalid="ignore", over="ignore"):
        s = (top.astype(np.float32) / np.float32(127)).astype(np.float64)
        s[bad] = np.nan
        q = np.divide(x, s[:, None], out=np.zeros_like(x), where=(s > 0)[:, None])
    return np.clip(np.rint(q), -127, 127).astype(np.int64), s


def rounding(y, dtype):
    """Half a step of `dtype` at y (subnormal steps included)."""
    if dtype == torch.float32:
        return np.abs(y) * EPS + 2.0 ** -150
    return np.abs(y) * 2.0 ** -11 + 2.0 ** -25


def swiglu(g, l, alpha=1.0, beta=0.0, limit=None):
    if limit is not None:
        g, l = np.minimum(g, limit), np.clip(l, -limit, limit)
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-alpha * g)) * (l + beta)


def product(a, sa, b, sb, bias=None, act="none", alpha=1.0, beta=0.0, limit=None):
    """Codes a [M, K], b [N, K] with scales -> (y, bound of the float32 steps before the last rounding), float64."""
    # whole numbers below 2^53: exact in any order
    t = (np.asarray(a, np.float64) @ np.asarray(b, np.float64).T) * np.asarray(sa, np.float64)[:, None] * np.asarray(sb, np.float64)
    y = t if bias is None else t + np.asarray(bias, np.float64)
    # the sum, two scales and the bias: three roundings of the term, one of the result
    err = 3 * EPS * np.abs(t) + EPS * np.abs(y) + 2.0 ** -148
    if act == "relu":
        y = np.where(y > 0, y, 0.0)
    elif act == "swiglu":
        g, l, dg, dl = y[:, 0::2], y[:, 1::2], err[:, 0::2], err[:, 1::2]
        y = swiglu(g, l, alpha, beta, limit)
        s = 1.0 / (1.0 + np.exp(np.minimum(-alpha * g, 700.0)))
        lin = np.abs(l) + abs(beta)
        # d/dg of g s(alpha g) is at most 1 + |alpha g| / 4; exp of a rounded argument is off by |alpha g| EPS, times
        # 1 - s in the quotient; eight roundings of expf (two steps), sum, quotient, sum and product
        err = dg * (1 + np.abs(alpha * g) * (1 - s)) * lin + np.abs(g) * s * (dl + EPS * lin) + np.abs(y) * EPS * (np.abs(alpha * g) * (1 - s) + 8) + 2.0 ** -148
    return y, 1.01 * err


def route(scores, k, normalize=True):
    """scores [T, E] -> (experts, weights float64, order, slots, offsets), and the weights' bound relative to them."""
    x = np.asarray(scores, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    T, E = x.shape
    experts = np.argsort(-x, axis=1, kind="stable")[:, :k]
    v = np.take_along_axis(x, experts, 1)
    weights, bound = np.zeros((T, k)), np.zeros((T, k))
    for t in range(T):
        if v[t, 0] == -np.inf:
            continue
        p, every = np.exp(v[t] - v[t, 0]), np.exp(x[t] - v[t, 0])
        weights[t] = p / (p.sum() if normalize else every.sum())
        # a difference rounded once, then exp within two steps, in both the number and the sum (whose terms weigh by
        # their size, at most exp(-d) d < 1 a step), up to 36 sums and the quotient
        d = np.where(np.isfinite(v[t]), v[t, 0] - v[t], 0.0)
        bound[t] = EPS * (d + 4 + 5 + 36 + 2)
    flat = experts.reshape(-1)
    order = np.argsort(flat, kind="stable")
    slots = np.empty_like(order)
    slots[order] = np.arange(len(order))
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=E))])
    return experts, weights, order, slots.reshape(T, k), offsets, bound


def close(got, want, err, dtype):
    """Whether every value of `got` lies within err, then one rounding to dtype, of `want`."""
    got = got.detach().cpu().double().numpy()
    assert got.shape == want.shape, (got.shape, want.shape)
    tol = err + rounding(np.abs(want) + err, dtype)
    limit = 65504.0 if dtype == torch.float16 else 3.4028235e38
    off = np.abs(got - want)
    fine = (off <= tol) | (np.isnan(got) & np.isnan(want)) | (~np.isfinite(got) & (np.abs(want) + tol >= limit) & (np.sign(got) == np.sign(want)))
    assert fine.all(), (int((~fine).sum()), float(np.nanmax(np.where(fine, 0, off / tol))), np.argwhere(~fine)[:4].tolist())
