"""AdamW with fp32 and 8-bit moments, every fp32 operation rounded by itself as the device does it, so that
results are compared bit for bit.  TEST INFRASTRUCTURE: imported by tests/ only."""
import numpy as np

F = np.float32
BLOCK = 256


def _power(x, t):
    y = 1.0
    while t:
        if t & 1:
            y *= x
        x *= x
        t >>= 1
    return y


def mix(x):
    with np.errstate(over="ignore"):
        x = np.asarray(x, np.uint32)
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x9E3779B9)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
        return x ^ (x >> np.uint32(16))


def _e4m3_values():
    """What the 256 bytes stand for."""
    out = np.zeros(256, np.float32)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)
        if e == 15 and m == 7:
            v = np.nan
        out[c] = -v if c & 128 else v
    return out


E4M3 = _e4m3_values()


def encode(x):
    """Bytes of values that e4m3 has."""
    up = np.searchsorted(E4M3[:127], np.abs(x)).astype(np.uint8)
    assert np.array_equal(E4M3[up], np.abs(x))
    return np.where(np.signbit(x), up | 128, up).astype(np.uint8)


def to_e4m3(q, bits):
    """q to one of its two neighbours, the upper one with the chance that sixteen bits give."""
    a = np.minimum(np.abs(q), F(448))
    low = a < F(2.0 ** -6)
    b = np.where(low, a + F(2.0 ** -6), a).astype(np.float32)
    c = ((b.view(np.uint32) + (bits.astype(np.uint32) << np.uint32(4))) & np.uint32(0xFFF00000)).view(np.float32)
    return np.where(low, c - F(2.0 ** -6), c).astype(np.float32)


def step(param, grad, state, t, hyper, decay=1.0, grad_scale=1.0, seed=0, counter=0):
    """The step number t (from 1 on) of one tensor; state is (m, v) or (m codes, v codes, m scales, v scales).
    Returns (param, state)."""
    lr, beta1, beta2, eps, wd = hyper
    size = F(lr / (1.0 - _power(beta1, t)))
    root = F(1.0 / np.sqrt(1.0 - _power(beta2, t)))
    keep = F(1) - F(decay) * F(lr * wd)
    n = param.size
    eight = len(state) == 4
    if eight:
        mc, vc, ms, vs = state
        at = np.arange(n) // BLOCK
        m = E4M3[mc] * ms[at]
        v = E4M3[vc] * vs[at]
        v = v * v
    else:
        m, v = state
    g = grad * F(grad_scale)
    m = m * F(beta1) + g * F(1.0 - beta1)
    v = v * F(beta2) + (g * g) * F(1.0 - beta2)
    r = np.sqrt(v)
    param = param * keep - (m / (r * root + F(eps))) * size
    assert param.dtype == m.dtype == v.dtype == np.float32
    if not eight:
        return param, (m, v)
    key = mix(np.uint32((seed + 0x9E3779B9 * t) & 0xFFFFFFFF))
    h = mix(((counter + np.arange(n, dtype=np.uint64)) & 0xFFFFFFFF).astype(np.uint32) ^ key)
    out = []
    for x, bits, is_root in ((m, h & np.uint32(0xFFFF), False), (r, h >> np.uint32(16), True)):
        blocks = -(-n // BLOCK)
        padded = np.zeros(blocks * BLOCK, np.float32)
        padded[:n] = np.abs(x)
        top = padded.reshape(blocks, BLOCK).max(1)
        live = top > F(2.0 ** -100)
        with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
            inverse = np.where(live, F(1) / top * F(448), F(0)).astype(np.float32)
        scale = np.where(live, top * (F(1) / F(448)), F(0)).astype(np.float32)
        q = x * inverse[at]
        c = to_e4m3(q, bits)
        if is_root:
            c = np.where((q > 0) & (c < F(2.0 ** -9)), F(2.0 ** -9), c).astype(np.float32)
        out.append((encode(np.copysign(c, q)), scale))
    return param, (out[0][0], out[1][0], out[0][1], out[1][1])
