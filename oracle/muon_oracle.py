"""The orthogonalised optimizer step in 64 bits, and how far rounding can carry it.  TEST INFRASTRUCTURE: imported by tests/ only."""
import numpy as np

A, B, C = 3.4445, -4.7750, 2.0315


def update(grad, mean, mu=0.95, eps=1e-7, nesterov=True, scale=1.0):
    """(u / (|u| + eps), the new mean)"""
    g = np.asarray(grad, np.float64) * scale
    mean = mu * np.asarray(mean, np.float64) + (1 - mu) * g
    u = (1 - mu) * g + mu * mean if nesterov else mean
    return u / (np.sqrt(np.sum(u * u)) + eps), mean


def orthogonal(x, steps=5, a=A, b=B, c=C):
    """The iteration, and the singular values of its operand before every step."""
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    found = []
    for _ in range(steps):
        found.append(np.linalg.svd(x, compute_uv=False))
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.T if tall else x), found


def reach(x, steps=5, a=A, b=B, c=C, unit=2.0 ** -24):
    """How far the computed result may be from the exact one, in the 2-norm of all values.

    A step is p(X) = a X + b A X + c A A X with A = X X^T.  A computed product P Q is off by at most `grow` units of |P| |Q|: the
    operands' two parts by two units each, the product of the small parts, which is left out, one, and 256 additions one behind
    another half of that.  In the 2-norm of all values |P| |Q| is at most the norm of P times that of Q; with size and top the
    norm and the largest singular value of X, and rows its shorter side, that makes the step's own error at most
    grow size (|a| + root(rows) (2 |b| top^2 + 4 |c| top^4)).  What a step makes of an error of its operand: the derivative of an
    odd matrix polynomial is in this norm at most the largest of |p'| and |p(s) / s| over the singular values."""
    if x.size == 0:
        return 0.0
    total, rows = 0.0, min(x.shape)
    grow = (5 + 128) * unit
    for s in orthogonal(x, steps, a, b, c)[1]:
        t = np.linspace(0, s.max() * (1 + 1e-3), 2001)
        slope = max(np.max(np.abs(a + 3 * b * t ** 2 + 5 * c * t ** 4)), np.max(np.abs(a + b * t ** 2 + c * t ** 4)))
        size, top = np.sqrt(np.sum(s * s)), s.max()
        own = grow * size * (abs(a) + np.sqrt(rows) * (2 * abs(b) * top ** 2 + 4 * abs(c) * top ** 4))
        total = slope * total + own
    return total
