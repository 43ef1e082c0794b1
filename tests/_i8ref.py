"""The 8-bit projections in 64 bits, written from their definitions: codes and scales of rows, products of codes."""
import numpy as np

HALF = 2.0 ** -24  # half a step of fp32, relative


def silu_mul(gu):
    k = gu.shape[1] // 2
    g, u = gu[:, :k].astype(np.float64), gu[:, k:].astype(np.float64)
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def quantize(t, factor=None):
    """Codes and scales of the rows t (float64), scales times factor (one a row)."""
    t = np.asarray(t, np.float64)
    top = np.abs(t).max(-1)
    scale = top / 127.0 * (1.0 if factor is None else factor)
    bad = ~np.isfinite(top) | (scale > np.finfo(np.float32).max)
    safe = np.where((top > 0) & ~bad, top, 1.0)
    codes = np.rint(np.where(bad[:, None], 0.0, t) * 127.0 / safe[:, None]).astype(np.int8)
    return codes, np.where(bad, np.nan, np.where(top > 0, scale, 0.0))


def rmsnorm(x, w=None, eps=1e-6):
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        factor = 1.0 / np.sqrt((x * x).mean(-1) + eps)
    return quantize(x if w is None else x * np.asarray(w, np.float64), factor)


def norm_tol(k):
    """Relative error of the norm's scale: the sum of squares adds at most 64 terms a thread, 6 steps of a wave and 16 waves in
    fp32, each half a step off; the root halves that; and the scale is rounded once."""
    return ((64 if k > 16384 else 16) + 6 + 16) / 2 * HALF + HALF


def product(q, s, w, ws):
    """Products of codes with scales, in 64 bits (the sums are whole numbers below 2^53: exact)."""
    return (q.astype(np.float64) @ w.astype(np.float64).T) * np.asarray(s, np.float64)[:, None] * np.asarray(ws, np.float64)


# the sum rounded to fp32 and two products, each half a step (their second-order terms are far below a tenth of one)
PRODUCT_TOL = 3.1 * HALF
