"""The operators in 8-bit integers from their definitions, in 64 bits (numpy), with bounds on what fp32 may change.

Half a step of bf16 is taken as 2^-8 of a value, one of fp32 as 2^-24."""
import numpy as np

HALF16, HALF32, TINY = 2.0 ** -8, 2.0 ** -24, 2.0 ** -134


def pitch(k):
    return -(-k // 16) * 16


def whole_numbers(u):
    """Rows as integers and the largest magnitude of each; a row with a NaN or an infinity is 0 with NaN."""
    u = np.asarray(u, np.float64)
    top = np.abs(u).max(-1)
    bad = ~np.isfinite(u).all(-1)
    safe = np.where(bad | (top == 0), 1.0, top)
    # 127 u and the largest magnitude are exact for bf16, and a quotient half way between two integers is one of fp64.
    q = np.rint(np.where(bad[..., None], 0.0, u) * 127.0 / safe[..., None])
    return q.astype(np.int8), np.where(bad, np.nan, top)


def norm(x, residual, weight, eps):
    """(x [+ residual], its RMSNorm times weight, a relative bound on the norm's values in fp32)."""
    v = x if residual is None else x + residual
    if weight is None:
        return v, v, 0.0
    k = v.shape[-1]
    u = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * weight
    # A sum of squares is a chain of at most 8 ceil(k / 2048) additions, then 8 more, all of positive numbers, of values
    # that are off by half a step each (two in the square); its root halves that. Beside it: the mean, eps, the root, the
    # reciprocal, and two products.
    chain = 8 * -(-k // 2048) + 8 + 2
    return v, u, (chain / 2 + 6 + 1) * HALF32


def product(x, residual, weight, eps, wq, ws, gated=False):
    """y in 64 bits and a bound on the error of a call's y, for tokens x [m, k] (float64), integers wq and scales ws."""
    v, u, off = norm(x, residual, weight, eps)
    q, top = whole_numbers(u)
    xs = top / 127.0
    acc = q.astype(np.float64) @ wq.astype(np.float64).T
    y = acc * xs[:, None] * ws
    size = np.abs(xs[:, None] * ws)
    # The scale: the largest value's error, and the division. The sum's rounding to fp32 and two products with scales.
    bound = np.abs(y) * (off + 4 * HALF32)
    if off:
        # An integer may be the next one where the quotient lies as near to a half as fp32 is off: u and the largest by
        # `off` of themselves, 127 u and the quotient by half a step.
        with np.errstate(invalid="ignore", divide="ignore"):
            t = np.nan_to_num(np.abs(u) * 127.0 / np.where(top > 0, top, 1.0)[:, None])
        unsure = np.abs(t - np.floor(t) - 0.5) <= 127.0 * (2 * off + 3 * HALF32)
        bound = bound + size * (unsure.astype(np.float64) @ np.abs(wq.astype(np.float64)).T)
    if gated:
        n = y.shape[1] // 2
        g, h, eg, eh = y[:, :n], y[:, n:], bound[:, :n], bound[:, n:]
        with np.errstate(over="ignore"):
            act = g / (1.0 + np.exp(-g))
        y = act * h
        # silu's slope is at most 1.1. Its exponential's argument is off by two half steps of 1.45 |g|, exponential and
        # reciprocal by a step each, the sum and the two products by half a step.
        bound = 1.1 * eg * (np.abs(h) + eh) + np.abs(act) * eh + np.abs(y) * (4 * np.abs(g) + 8) * HALF32
    return y, bound + (np.abs(y) + bound) * HALF16 + TINY


def residual_of(x, residual):
    """x + residual in float32, as stored before it is rounded to bf16."""
    return (x + residual).astype(np.float32)
