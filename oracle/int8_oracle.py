"""64-bit restatements of the int8 operators and of the token sort with its gradients (numpy),
written from their definitions; used by tests only."""
from __future__ import annotations

import numpy as np


def quantize_int8(x: np.ndarray) -> tuple:
    """``x`` float64 [rows, cols] -> (codes int8, scales float64): nearest code of the exact
    quotient 127 x / max|x|, ties to even."""
    x = np.asarray(x, dtype=np.float64)
    rows = x.shape[0]
    codes = np.zeros(x.shape, dtype=np.int8)
    scales = np.zeros(rows)
    for r in range(rows):
        if not np.all(np.isfinite(x[r])):
            scales[r] = np.nan
            continue
        amax = np.abs(x[r]).max()
        scales[r] = amax / 127.0
        if amax > 0:
            # 127 x is exact for 16-bit x; a quotient that is a tie is exact as well, and one that
            # is not is far further from a tie than the rounding of the division.
            codes[r] = np.rint(127.0 * x[r] / amax)
    return codes, scales


def product(a, a_scale, b, b_scale, bias=None) -> np.ndarray:
    """a_scale[m] b_scale[n] sum_k a[m,k] b[n,k] (+ bias[n]); the sums are exact in float64."""
    acc = np.asarray(a, np.float64) @ np.asarray(b, np.float64).T
    out = acc * np.asarray(a_scale, np.float64)[:, None] * np.asarray(b_scale, np.float64)[None, :]
    return out if bias is None else out + np.asarray(bias, np.float64)[None, :]


def silu(g: np.ndarray) -> np.ndarray:
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))


def dispatch(x, dest, rows: int, topk: int) -> np.ndarray:
    y = np.zeros((rows, x.shape[1]))
    for p, d in enumerate(dest):
        if 0 <= d < rows:
            y[d] = x[p // topk]
    return y


def combine(y, dest, weights, tokens: int, topk: int) -> np.ndarray:
    out = np.zeros((tokens, y.shape[1]))
    for p, d in enumerate(dest):
        if 0 <= d < y.shape[0]:
            w = 1.0 if weights is None else weights[p // topk, p % topk]
            out[p // topk] += w * y[d]
    return out


def combine_backward(grad, y, dest, weights, topk: int) -> tuple:
    gy = np.zeros_like(y, dtype=np.float64)
    gw = np.zeros((grad.shape[0], topk))
    for p, d in enumerate(dest):
        if 0 <= d < y.shape[0]:
            t, j = divmod(p, topk)
            gy[d] = (1.0 if weights is None else weights[t, j]) * grad[t]
            gw[t, j] = np.dot(grad[t], y[d])
    return gy, gw
