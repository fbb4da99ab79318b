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


UNIT = 2.0 ** -24


def _off(p, q, rng):
    """A product of computed operands, off as the kernel's may be: a value of an operand is two fp16 parts of 22 bits (2 units of itself,
    and 2^-40 of the largest possible one, where fp16 ends), what is left out of the products of parts (4 units) counts with
    them; 12 sums of 16 products a block of 64, each cut down to fp32, lose up to 12 units of what they hold, and the blocks'
    sums are added in fp32: a unit each, in any direction, the root of their number in all; and the result is rounded."""
    sign = lambda x: rng.integers(0, 2, x.shape) * 2.0 - 1.0  # noqa: E731
    p, q = p * (1 + 4 * UNIT * sign(p)), q * (1 + 4 * UNIT * sign(q))
    found = p @ q
    size = np.maximum(np.abs(found), np.sqrt((p * p) @ (q * q)))
    return found - 12 * UNIT * size * np.sign(found) + (1 + np.sqrt(p.shape[1] / 64)) * UNIT * size * sign(found)


def spread(x, steps=5, a=A, b=B, c=C, samples=4):
    """How far the computed result is from the exact one where every rounding is as large as it can be and its sign is a matter of
    chance: the largest of some samples, in the 2-norm of all values.  (A bound on every choice of signs, `reach`, is thousands of times
    as much, and would let results through that are off by 2^-12.)"""
    x = np.asarray(x.T if x.shape[0] > x.shape[1] else x, np.float64)
    want = orthogonal(x, steps, a, b, c)[0]
    worst = 0.0
    for k in range(samples):
        rng = np.random.default_rng(k)
        # u: three roundings, the factor and the product with it
        y = x * (1 + 5 * UNIT * (rng.integers(0, 2, x.shape) * 2.0 - 1.0))
        for _ in range(steps):
            s = _off(y, y.T, rng)
            s = (s + s.T) / 2
            t = b * s + c * _off(s, s, rng)
            y = _off(t + a * np.eye(len(t)), y, rng)
        worst = max(worst, float(np.sqrt(np.sum((y - want) ** 2))))
    return worst


def emulated(x, steps=5, a=A, b=B, c=C, parts=2, products=3):
    """The iteration with operands of fp16 parts and as many of the products of parts, sums in 64 bits: what two parts and three products
    are worth, and what fewer would be."""
    tall = x.shape[0] > x.shape[1]
    y, top = (x.T if tall else x).astype(np.float32), 1.0

    def split(v, most):
        up = 2.0 ** np.floor(np.log2(60000 / (1.01 * most)))
        hi = (v * up).astype(np.float16)
        lo = (v * up - hi.astype(np.float64)).astype(np.float16)
        return hi.astype(np.float64) / up, (lo.astype(np.float64) / up if parts == 2 else 0.0 * v)

    def product(p, q):
        return (p[0] @ q[0] + p[0] @ q[1] + (p[1] @ q[0] if products == 3 else 0.0)).astype(np.float32).astype(np.float64)
    grid = np.linspace(0, 1, 2001)
    for _ in range(steps):
        s = grid * top
        factor, following = np.max(np.abs(a + b * s ** 2 + c * s ** 4)), np.max(np.abs(a * s + b * s ** 3 + c * s ** 5))
        x2 = split(y, top)
        g = product(x2, (x2[0].T, x2[1].T))
        g = np.triu(g) + np.triu(g, 1).T
        g2 = split(g, top * top)
        t = a * np.eye(len(g)) + b * g + c * product(g2, g2)
        y, top = product(split(t, factor), x2), 1.001 * following
    return y.T if tall else y
