"""Plain 64-bit forms of the block-scaled operators, for the tests: numpy only,
written from the definitions."""
import math

import numpy as np


def exponents(x, block_rows=1):
    """Integer exponents of the blocks of x [R, C]: [ceil(R / block_rows), ceil(C / 128)]."""
    x = np.asarray(x, np.float64)
    R, C = x.shape
    out = np.zeros((-(-R // block_rows), -(-C // 128)), np.int64)
    for i in range(out.shape[0]):
        for j in range(out.shape[1]):
            b = np.abs(x[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128])
            b = b[np.isfinite(b)]
            top = b.max() if b.size else 0.0
            if top == 0.0:
                continue
            p = math.frexp(top)[1] - 10          # 448 * 2^p is below top here
            while top > 448.0 * 2.0 ** p:
                p += 1
            out[i, j] = max(p, -126)
    return out


def spread(e, shape, block_rows=1):
    """Exponents per element."""
    R, C = shape
    return np.repeat(np.repeat(e, block_rows, 0)[:R], 128, 1)[:, :C]


def round_e4m3(v):
    """Nearest E4M3 value (ties to even) of |v| <= 448; NaN for NaN and infinities."""
    v = np.asarray(v, np.float64)
    a = np.abs(v)
    bad = ~np.isfinite(a)
    a = np.where(bad, 1.0, a)
    e = np.maximum(np.frexp(a)[1] - 1, -6)
    q = np.exp2(e - 3.0)
    r = np.rint(a / q) * q
    return np.where(bad, np.nan, np.copysign(r, v))


def cast(x, block_rows=1):
    """(values on the scaled E4M3 grid, exponents per element)."""
    e = spread(exponents(x, block_rows), np.shape(x), block_rows)
    s = np.exp2(e.astype(np.float64))
    return round_e4m3(np.asarray(x, np.float64) / s) * s, e


def norm(r, gamma, eps):
    r = np.asarray(r, np.float64)
    rstd = 1.0 / np.sqrt((r * r).mean(1, keepdims=True) + eps)
    return r * rstd * np.asarray(gamma, np.float64), rstd


def norm_backward(r, gamma, eps, dy, dr=None):
    r, gamma, dy = (np.asarray(t, np.float64) for t in (r, gamma, dy))
    rstd = 1.0 / np.sqrt((r * r).mean(1, keepdims=True) + eps)
    hat = r * rstd
    g = gamma * dy
    dx = rstd * (g - hat * (g * hat).mean(1, keepdims=True))
    if dr is not None:
        dx = dx + np.asarray(dr, np.float64)
    return dx, (dy * hat).sum(0)
