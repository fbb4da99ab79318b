"""Rotation of heads by position, norms of heads and their gradients in 64 bits, with what each value's terms add up to in
absolute value -- the measure that rounding errors go by.  TEST INFRASTRUCTURE: imported by tests/ only."""
import math

import numpy as np


def frequencies(d, base=10000.0, scaling="none", factor=1.0, original=1.0, low=1.0, high=32.0):
    """Radians a position of each of d / 2 pairs."""
    if scaling == "base" and d > 2:
        base = base * factor ** (d / (d - 2))
    f = np.array([base ** (-2.0 * i / d) for i in range(d // 2)])
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        keep = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
        f = keep * f + (1 - keep) * f / factor
    return f


def angles(positions, turns):
    """Radians [rows][pairs] of whole positions, in the whole numbers that the frequencies are."""
    with np.errstate(over="ignore"):
        phase = np.asarray(positions, np.int64).astype(np.uint64)[:, None] * np.asarray(turns).astype(np.uint64)[None, :]
    return phase.astype(np.int64).astype(np.float64) * (2 * math.pi / 2.0 ** 64)


def places(d, interleaved):
    """(first, second) features of the pairs of d features."""
    i = np.arange(d // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + d // 2)


def rotate(x, angle, d, interleaved, amplitude=1.0, inverse=False):
    """x [rows][heads][D] turned, and what the terms of each value add up to in absolute value."""
    x = np.asarray(x, np.float64)
    out, size = x.copy(), np.abs(x)
    if d:
        a, b = places(d, interleaved)
        c, s = amplitude * np.cos(angle)[:, None], amplitude * np.sin(angle)[:, None] * (-1 if inverse else 1)
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        both = abs(amplitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
        size[..., a] = size[..., b] = both
    return out, size


def forward(x, w, eps, angle, d, interleaved, amplitude=1.0):
    """(out, rstd, size of out)"""
    x = np.asarray(x, np.float64)
    rstd = 1.0 / np.sqrt(np.mean(x * x, axis=2) + eps)
    y = x * rstd[..., None] * (1.0 if w is None else np.asarray(w, np.float64))
    out, size = rotate(y, angle, d, interleaved, amplitude)
    return out, rstd, size


def backward(d_out, x, w, rstd, angle, d, interleaved, amplitude=1.0):
    """(d_x, d_weight, size of d_x, size of d_weight), at the given rstd."""
    x = np.asarray(x, np.float64)
    w = 1.0 if w is None else np.asarray(w, np.float64)
    g, size = rotate(d_out, angle, d, interleaved, amplitude, inverse=True)
    r = np.asarray(rstd, np.float64)[..., None]
    xhat = x * r
    wd = g * w
    dx = r * (wd - xhat * np.mean(wd * xhat, axis=2, keepdims=True))
    big = size * np.abs(w)
    dx_size = r * (big + np.abs(xhat) * np.mean(big * np.abs(xhat), axis=2, keepdims=True))
    return dx, np.sum(g * xhat, axis=(0, 1)), dx_size, np.sum(size * np.abs(xhat), axis=(0, 1))
