"""The 8-bit operators from their definitions in 64 bits, on the host: what tests/test_gpu_i8.py and test_gpu_moe8.py compare
with, and how far the kernels may be from it. u = 2^-24 is half a step of fp32."""
import numpy as np
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LOWEST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half the smallest step


def rows8(x):
    """(q, a) of the rows of x [M, K]: whole numbers as float64 and the rows' largest magnitudes. 127 x is exact in 64 bits for a
    32-bit x, and so is a tie of the quotient; a quotient that is no tie is at least 2^-33 (relative) off one. A row with a
    NaN or an infinity: q = 0, a = NaN"""
    x = x.double().cpu().numpy()
    a = np.max(np.abs(x), axis=1, keepdims=True)
    bad = ~np.isfinite(x).all(axis=1, keepdims=True)
    with np.errstate(all="ignore"):
        q = np.rint(127.0 * x / np.where(a > 0, a, 1.0))
    return np.where(bad, 0.0, q), np.where(bad, np.nan, a)


def product(q, a, w, ws):
    """q [M, K] and row magnitudes a [M, 1] through int8 w [N, K] with channel scales ws [N]"""
    return (q @ w.double().cpu().numpy().T) * (a / 127.0) * ws.double().cpu().numpy()[None, :]


def product_bound(p, y, dtype):
    """of y = p (+ bias) in `dtype`: p is the integer sum (exact) cast to fp32, times a scale that is a rounded quotient, times
    another: four roundings, (1 + u)^4 - 1 < 4.01 u; the bias adds one of y, the type its half step"""
    h, low = HALF[dtype], LOWEST[dtype]
    return 4.01 * U * np.abs(p) * (1 + 2 * h) + (U + h) * 1.01 * np.abs(y) + low + 2.0 ** -148


def mlp(q, a, wg, wu, wd, sg, su, sd):
    """(y, slack, size): the gated MLP in 64 bits, how far y may move because a gated value that lies within its own error of a
    border between two whole numbers may be rounded to the other one, and the sum of its terms' magnitudes.

    The error of h = silu(g) u, relative: g and u carry 4 u each; silu'(g) g / silu(g) = 1 + g (1 - sigmoid(g)) is at most
    1 + |g| in size; e^-g by exp2 of a rounded product carries (|g| + 2) u, counted twice for the hardware's exp2; the sum,
    the quotient and the product round once each: (4 (1 + |g|) + 2 (|g| + 2) + 3 + 4) u < (16 + 6 |g|) u. The row's largest
    value carries as much, the quotient to whole numbers 3 u more."""
    g, v = product(q, a, wg, sg), product(q, a, wu, su)
    with np.errstate(over="ignore"):
        h = g / (1.0 + np.exp(-g)) * v
    top = np.max(np.abs(h), axis=1, keepdims=True)
    level = 127.0 * h / np.where(top > 0, top, 1.0)
    err = (2 * (16 + 6 * np.max(np.abs(g), axis=1, keepdims=True)) + 3) * U
    p = np.rint(level)
    near = np.abs(np.abs(level - np.floor(level)) - 0.5) <= err * np.maximum(np.abs(level), 0.5)
    sdn = sd.double().cpu().numpy()[None, :]
    wn = wd.double().cpu().numpy()
    y = (p @ wn.T) * (top / 127.0) * sdn
    # with moved = y + (what the other roundings add) the kernel gives moved (1 + e)(1 + 4.01 u), e <= err / 2 the error of the
    # row's largest value: at most |moved - y| (1 + err) + err |y| from y (4.01 u < err / 2; the roundings of y's own product
    # are product_bound's)
    slack = (near.astype(np.float64) @ np.abs(wn).T) * (top / 127.0) * np.abs(sdn) * (1 + err) + err * np.abs(y)
    return y, slack, (np.abs(p) @ np.abs(wn).T) * (top / 127.0) * np.abs(sdn)
