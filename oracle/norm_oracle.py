"""The edge between two blocks of a residual network and its gradients in 64 bits, with what each value's
terms add up to in absolute value -- the measure that rounding errors of a sum go by.  TEST INFRASTRUCTURE:
imported by tests/ only."""
import numpy as np


def forward(residual, block=None, gate=None, post=None, pre=None, a=1.0, eps=1e-6):
    """dict of stream, out, block_rstd, stream_rstd, and `size` of stream and out.  gate broadcasts."""
    r = np.asarray(residual, np.float64)
    found, size = {}, {}
    x, big = r, np.abs(r)
    if block is not None:
        u = np.asarray(block, np.float64)
        y = u
        if post is not None:
            rho = 1.0 / np.sqrt(np.mean(u * u, axis=1, keepdims=True) + eps)
            found["block_rstd"] = rho[:, 0]
            y = u * rho * np.asarray(post, np.float64)
        if gate is not None:
            y = y * np.asarray(gate, np.float64)
        x, big = a * r + y, np.abs(a * r) + np.abs(y)
        found["stream"], size["stream"] = x, big
    rho = 1.0 / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + eps)
    found["stream_rstd"] = rho[:, 0]
    if pre is not None:
        w = np.asarray(pre, np.float64)
        found["out"], size["out"] = x * rho * w, big * rho * np.abs(w)
    return found, size


def _through(d, big, x, rho, w):
    """(gradient of x, its size, gradient of w, its size) where y = x rho w and d is y's gradient."""
    xh = x * rho
    dx = d * w
    mean = np.mean(dx * xh, axis=1, keepdims=True)
    mean_size = np.mean(big * np.abs(w * xh), axis=1, keepdims=True)
    return (rho * (dx - xh * mean), rho * (big * np.abs(w) + np.abs(xh) * mean_size),
            np.sum(d * xh, axis=0), np.sum(big * np.abs(xh), axis=0))


def backward(stream, stream_rstd=None, d_out=None, d_stream=None, block=None, block_rstd=None, gate=None,
             post=None, pre=None, a=1.0):
    """Gradients (and sizes) of residual, block, gate, post, pre at the stored stream and rstd's."""
    f = lambda v: None if v is None else np.asarray(v, np.float64)  # noqa: E731
    x, d_out, d_stream, u, gate, post, pre = [f(v) for v in (stream, d_out, d_stream, block, gate, post, pre)]
    found, size = {}, {}
    t = np.zeros_like(x) if d_stream is None else d_stream
    big = np.abs(t)
    if pre is not None:
        dx, dx_size, found["pre"], size["pre"] = _through(d_out, np.abs(d_out), x, f(stream_rstd)[:, None], pre)
        t, big = t + dx, big + dx_size
    found["residual"], size["residual"] = a * t, np.abs(a) * big
    if u is not None:
        rho = None if post is None else f(block_rstd)[:, None]
        y = u if post is None else u * rho * post
        if gate is not None:
            g, g_size = t * y, big * np.abs(y)
            for axis in (0, 1):
                if gate.shape[axis] == 1 and g.shape[axis] != 1:
                    g, g_size = g.sum(axis, keepdims=True), g_size.sum(axis, keepdims=True)
            found["gate"], size["gate"] = g.reshape(gate.shape), g_size.reshape(gate.shape)
            t, big = t * gate, big * np.abs(gate)
        if post is not None:
            t, big, found["post"], size["post"] = _through(t, big, u, rho, post)
        found["block"], size["block"] = t, big
    return found, size
