"""The norms between two blocks with gate and residual scale, and their gradients, through the C ABI, against 64
bits.  A result is a sum (of squares over a row, of rows for a weight) in fp32 and a few products: each addition and
product rounds by half a step of what the terms add up to in absolute value."""
import ctypes

import numpy as np
import pytest

from oracle import norm_oracle as no

HALF = 2.0 ** -24
GATES = {"none": 0, "feature": 1, "row": 2, "full": 3}


def _gate_shape(kind, rows, F):
    return {"none": None, "feature": (1, F), "row": (rows, 1), "full": (rows, F)}[kind]


def _case(rows, F, gate="none", block=True, post=True, pre=True, seed=0, spread=1.0):
    rng = np.random.RandomState(seed + rows + F)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    c = dict(residual=f(rows, F) * np.float32(spread), a=1.0, block=None, gate=None, post=None, pre=1 + f(F) * np.float32(0.3) if pre else None)
    if block:
        c.update(a=float(np.float32(0.7)), block=f(rows, F) * np.float32(2), post=1 + f(F) * np.float32(0.3) if post else None)
        shape = _gate_shape(gate, rows, F)
        c["gate"] = None if shape is None else f(*shape)
    return c


class _Memory(object):
    """Rows of a device tensor with a stride and a start of their own, in a sea of marks."""
    MARK = -77.0

    def __init__(self, value, pad=0, offset=0):
        import torch
        value = np.asarray(value, np.float32)
        self.rows, self.F = value.shape
        self.stride = self.F + pad
        self.all = torch.full((self.rows * self.stride + offset + 8,), self.MARK, device="cuda")
        self.offset = offset
        self.t = torch.as_strided(self.all, value.shape, (self.stride, 1), offset)
        self.t.copy_(torch.from_numpy(value))
        self.ptr = self.all.data_ptr() + 4 * offset

    def intact(self):
        import torch
        seen = torch.ones_like(self.all, dtype=torch.bool)
        torch.as_strided(seen, (self.rows, self.F), (self.stride, 1), self.offset).fill_(False)
        return bool((self.all[seen] == self.MARK).all())


def _vec(v):
    import torch
    return None if v is None else torch.from_numpy(np.ascontiguousarray(v, dtype=np.float32)).cuda()


def _at(x):
    return None if x is None else x.ptr if isinstance(x, _Memory) else x.data_ptr()


def _args(c, gate, mem, vecs, rows, F):
    from ngraph_python_b200 import lib
    a = lib.NormArgs()
    a.rows, a.features, a.gate_kind, a.residual_scale, a.eps = rows, F, GATES[gate], c["a"], 1e-6
    for name in ("block", "residual", "stream", "out"):
        m = mem.get(name)
        setattr(a, name, _at(m))
        setattr(a, name + "_stride", m.stride if m is not None else 0)
    g = mem.get("gate")
    a.gate = _at(g if g is not None else vecs.get("gate"))
    a.gate_stride = g.stride if g is not None else 0
    a.post_weight, a.pre_weight = _at(vecs["post"]), _at(vecs["pre"])
    a.block_rstd, a.stream_rstd = _at(vecs.get("block_rstd")), _at(vecs.get("stream_rstd"))
    return a


def _forward(c, gate, pad=0, offset=0, in_place=False, keep=True):
    import torch
    from ngraph_python_b200 import lib
    rows, F = c["residual"].shape
    mem = dict(residual=_Memory(c["residual"], pad, offset))
    vecs = dict(post=_vec(c["post"]), pre=_vec(c["pre"]))
    if c["block"] is not None:
        mem["block"] = _Memory(c["block"], 2 * pad, offset)
        mem["stream"] = mem["residual"] if in_place else _Memory(np.zeros((rows, F)), 3 * pad, offset)
    if c["gate"] is not None:
        if gate == "full":
            mem["gate"] = _Memory(c["gate"], pad, offset)
        else:
            vecs["gate"] = _vec(c["gate"])
    if c["pre"] is not None:
        mem["out"] = _Memory(np.zeros((rows, F)), pad, offset)
    if keep:
        vecs["stream_rstd"] = torch.zeros((rows,), device="cuda")
        if c["post"] is not None:
            vecs["block_rstd"] = torch.zeros((rows,), device="cuda")
    a = _args(c, gate, mem, vecs, rows, F)
    lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), 0))
    torch.cuda.synchronize()
    assert all(m.intact() for m in mem.values())
    got = {k: mem[k].t.cpu().numpy() for k in ("stream", "out") if k in mem}
    got.update({k: vecs[k].cpu().numpy() for k in ("stream_rstd", "block_rstd") if k in vecs})
    return got, (a, mem, vecs)


def _check_forward(got, c, F):
    want, size = no.forward(c["residual"], c["block"], c["gate"], c["post"], c["pre"], c["a"], 1e-6)
    # a mean of squares: at most F / 32 additions one after another and a tree, whatever the threads; half of its
    # error goes into the root, and twelve roundings stand for the products
    steps = F / 32 + 24
    for k, v in got.items():
        s = size.get(k, np.abs(want[k]))
        assert np.all(np.abs(v - want[k]) <= steps * HALF * s), k


FORWARD = [(rows, F, gate, block, post, pre)
           for rows, F in ((1, 1), (3, 5), (1, 2048), (33, 64), (7, 1001), (300, 256), (2, 4096), (5, 8192), (2, 20000), (1000, 100), (3, 16388))
           for gate, block, post, pre in (("feature", True, True, True), ("row", True, True, True), ("full", True, True, True),
                                          ("none", True, False, True), ("full", True, False, False), ("none", True, True, False),
                                          ("none", False, False, True))]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,F,gate,block,post,pre", FORWARD)
def test_forward(rows, F, gate, block, post, pre):
    c = _case(rows, F, gate, block, post, pre)
    got, _ = _forward(c, gate)
    assert set(got) == {"stream_rstd"} | ({"stream"} if block else set()) | ({"out"} if pre else set()) | ({"block_rstd"} if post else set())
    _check_forward(got, c, F)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,F,pad,offset", [(9, 96, 4, 0), (9, 96, 1, 0), (9, 96, 0, 1), (6, 515, 5, 3), (4, 6000, 2, 0), (3, 9000, 8, 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_forward_strides(rows, F, pad, offset, in_place):
    """Rows apart, starts off 16 bytes, the stream in place of the residual, and nothing kept for gradients."""
    c = _case(rows, F, "full")
    got, _ = _forward(c, "full", pad, offset, in_place, keep=False)
    _check_forward(got, c, F)


def _backward(c, gate, x, rstd, rho, d_out, d_stream, pad=0, offset=0, in_place=False, leave_out=()):
    import torch
    from ngraph_python_b200 import lib
    rows, F = c["residual"].shape
    mem = {}
    vecs = dict(post=_vec(c["post"]), pre=_vec(c["pre"]), stream_rstd=_vec(rstd), block_rstd=_vec(rho))
    if c["block"] is not None:
        mem["block"], mem["stream"] = _Memory(c["block"], pad, offset), _Memory(x, 2 * pad, offset)
    else:
        mem["residual"] = _Memory(x, pad, offset)
    if c["gate"] is not None:
        if gate == "full":
            mem["gate"] = _Memory(c["gate"], pad, offset)
        else:
            vecs["gate"] = _vec(c["gate"])
    a = _args(c, gate, mem, vecs, rows, F)
    d = lib.NormGrads()
    ends = dict(d_out=None if d_out is None else _Memory(d_out, pad, offset), d_stream=None if d_stream is None else _Memory(d_stream, 2 * pad, offset))
    ends["d_residual"] = ends["d_stream"] if in_place else _Memory(np.full((rows, F), 5.0), pad, offset)
    if c["block"] is not None:
        ends["d_block"] = _Memory(np.full((rows, F), 5.0), 3 * pad, offset)
    if gate == "full":
        ends["d_gate"] = _Memory(np.full((rows, F), 5.0), pad, offset)
    sums = {}
    if gate in ("feature", "row"):
        sums["d_gate"] = torch.full((c["gate"].size,), 5.0, device="cuda")
    for name in ("post", "pre"):
        if c[name] is not None:
            sums["d_%s_weight" % name] = torch.full((F,), 5.0, device="cuda")
    for name in leave_out:
        ends.pop(name, None)
        sums.pop(name, None)
    for k, m in ends.items():
        setattr(d, k, _at(m))
        setattr(d, k + "_stride", m.stride if m is not None else 0)
    for k, v in sums.items():
        setattr(d, k, v.data_ptr())
    nbytes = lib.norm_bprop_scratch_bytes(a)
    scratch = torch.full((nbytes,), 0xA5, dtype=torch.uint8, device="cuda")
    lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch.data_ptr(), nbytes, 0))
    torch.cuda.synchronize()
    assert all(m is None or m.intact() for m in list(mem.values()) + list(ends.values()))
    names = dict(d_residual="residual", d_block="block", d_gate="gate", d_post_weight="post", d_pre_weight="pre")
    return {names[k]: (v.t if isinstance(v, _Memory) else v).cpu().numpy() for k, v in list(ends.items()) + list(sums.items()) if k in names}


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["feature", "row", "full"])
@pytest.mark.parametrize("rows,F,pad", [(5000, 37, 0), (900, 1001, 0), (2400, 99, 2), (400, 4099, 0), (700, 2050, 3), (3000, 61, 3)])
def test_many_ragged_rows(rows, F, pad, gate):
    """More rows than blocks, each begun elsewhere within sixteen bytes."""
    c = _case(rows, F, gate)
    got, _ = _forward(c, gate) if not pad else _forward_alike(c, gate, pad)
    _check_forward(got, c, F)
    rng = np.random.RandomState(9)
    x, rstd, rho = _stored(c)
    d = [rng.standard_normal((rows, F)).astype(np.float32) for _ in range(2)]
    _check_backward(_backward(c, gate, x, rstd, rho, *d), c, x, rstd, rho, *d)


@pytest.mark.gpu
@pytest.mark.parametrize("F", [3407, 4053, 4091, 4093, 4095, 4097, 8189, 8190, 8191, 8193, 16381, 16382, 16383])
def test_ragged_rows_around_the_limits_of_shared_memory(F):
    for rows in (2, 400):
        c = _case(rows, F, "feature")
        got, _ = _forward(c, "feature")
        _check_forward(got, c, F)
    if F < 9000:
        rng = np.random.RandomState(9)
        x, rstd, rho = _stored(c)
        d = [rng.standard_normal((rows, F)).astype(np.float32) for _ in range(2)]
        _check_backward(_backward(c, "feature", x, rstd, rho, *d), c, x, rstd, rho, *d)


def _forward_alike(c, gate, pad):
    """All rows `pad` apart."""
    import torch
    from ngraph_python_b200 import lib
    rows, F = c["residual"].shape
    mem = {k: _Memory(v, pad) for k, v in dict(residual=c["residual"], block=c["block"], stream=np.zeros((rows, F)), out=np.zeros((rows, F))).items()}
    vecs = dict(post=_vec(c["post"]), pre=_vec(c["pre"]))
    if gate == "full":
        mem["gate"] = _Memory(c["gate"], pad)
    else:
        vecs["gate"] = _vec(c["gate"])
    lib.check(lib.raw().b2_norm_fprop(ctypes.byref(_args(c, gate, mem, vecs, rows, F)), 0))
    torch.cuda.synchronize()
    assert all(m.intact() for m in mem.values())
    return {k: mem[k].t.cpu().numpy() for k in ("stream", "out")}, None


def _stored(c):
    """What a forward pass leaves, in fp32."""
    want, _ = no.forward(c["residual"], c["block"], c["gate"], c["post"], c["pre"], c["a"], 1e-6)
    x = want.get("stream", c["residual"]).astype(np.float32)
    rstd = (1 / np.sqrt(np.mean(x.astype(np.float64) ** 2, axis=1) + 1e-6)).astype(np.float32)
    return x, rstd, None if c["post"] is None else want["block_rstd"].astype(np.float32)


def _check_backward(got, c, x, rstd, rho, d_out, d_stream):
    rows, F = x.shape
    want, size = no.backward(x, rstd, d_out, d_stream, c["block"], rho, c["gate"], c["post"], c["pre"], c["a"])
    # rows: two means one after the other; columns: sums over the rows, of values that have a row's errors
    of_row = 2 * (F / 32 + 24)
    for k, v in got.items():
        w, s = want[k].reshape(v.shape), size[k].reshape(v.shape)
        steps = of_row + (rows + 16 if k in ("post", "pre", "gate") else 0)
        assert np.all(np.abs(v - w) <= steps * HALF * s), k


@pytest.mark.gpu
@pytest.mark.parametrize("rows,F,gate,block,post,pre", FORWARD)
def test_backward(rows, F, gate, block, post, pre):
    c = _case(rows, F, gate, block, post, pre)
    rng = np.random.RandomState(5)
    x, rstd, rho = _stored(c)
    d_out = rng.standard_normal((rows, F)).astype(np.float32) if pre else None
    d_stream = rng.standard_normal((rows, F)).astype(np.float32)
    got = _backward(c, gate, x, rstd, rho, d_out, d_stream)
    assert set(got) == {"residual"} | ({"block"} if block else set()) | ({"gate"} if gate != "none" else set()) | \
        ({"post"} if post else set()) | ({"pre"} if pre else set())
    _check_backward(got, c, x, rstd, rho, d_out, d_stream)
    again = _backward(c, gate, x, rstd, rho, d_out, d_stream)
    assert all(np.array_equal(got[k], again[k]) for k in got)
    if pre:
        got = _backward(c, gate, x, rstd, rho, d_out, None)
        _check_backward(got, c, x, rstd, rho, d_out, None)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,F,pad,offset", [(9, 96, 4, 0), (700, 96, 1, 0), (9, 96, 0, 1), (6, 515, 5, 3), (4, 6000, 2, 0), (3, 9000, 8, 4)])
def test_backward_strides(rows, F, pad, offset):
    c = _case(rows, F, "full")
    rng = np.random.RandomState(6)
    x, rstd, rho = _stored(c)
    d_out, d_stream = [rng.standard_normal((rows, F)).astype(np.float32) for _ in range(2)]
    for in_place in (False, True):
        _check_backward(_backward(c, "full", x, rstd, rho, d_out, d_stream, pad, offset, in_place), c, x, rstd, rho, d_out, d_stream)


@pytest.mark.gpu
@pytest.mark.parametrize("gate,post", [("feature", True), ("row", True), ("full", True), ("full", False), ("none", False)])
@pytest.mark.parametrize("rows,F,pad,offset", [(470, 5116, 0, 0), (470, 5120, 4, 4), (310, 5124, 0, 0), (310, 5119, 2, 1), (310, 6141, 1, 3), (450, 6144, 0, 0),
                                               (200, 8189, 0, 0), (200, 8189, 3, 2), (200, 8190, 2, 0), (200, 8192, 0, 0)])
def test_backward_of_long_rows(rows, F, pad, offset, gate, post):
    """Where a thread's share of a row, and the place of its weights, changes: two and more rows to a CTA, one behind another."""
    c = _case(rows, F, gate, True, post)
    rng = np.random.RandomState(8)
    x, rstd, rho = _stored(c)
    d_out, d_stream = [rng.standard_normal((rows, F)).astype(np.float32) for _ in range(2)]
    _check_backward(_backward(c, gate, x, rstd, rho, d_out, d_stream, pad, offset), c, x, rstd, rho, d_out, d_stream)


@pytest.mark.gpu
@pytest.mark.parametrize("gate,block", [("feature", True), ("full", True), ("none", True), ("none", False)])
@pytest.mark.parametrize("rows,F", [(3000, 64), (1600, 707), (1000, 1536), (1000, 1792), (700, 2047), (700, 2048), (500, 2560), (500, 3501), (400, 4096)])
def test_backward_of_many_rows(rows, F, gate, block):
    """More rows than CTAs, of all numbers of CTAs to an SM."""
    c = _case(rows, F, gate, block, block)
    rng = np.random.RandomState(9)
    x, rstd, rho = _stored(c)
    d_out, d_stream = [rng.standard_normal((rows, F)).astype(np.float32) for _ in range(2)]
    got = _backward(c, gate, x, rstd, rho, d_out, d_stream)
    _check_backward(got, c, x, rstd, rho, d_out, d_stream)
    again = _backward(c, gate, x, rstd, rho, d_out, d_stream)
    assert all(np.array_equal(got[k], again[k]) for k in got)


@pytest.mark.gpu
@pytest.mark.parametrize("gate,block", [("feature", True), ("row", True), ("full", True), ("none", False)])
@pytest.mark.parametrize("rows,F", [(12000, 4), (12000, 64), (12000, 101), (11000, 256), (10000, 260), (10000, 509), (10000, 512), (10000, 516)])
def test_forward_of_many_short_rows(rows, F, gate, block):
    c = _case(rows, F, gate, block, block)
    got, _ = _forward(c, gate)
    _check_forward(got, c, F)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["feature", "row", "full"])
def test_backward_of_some(gate):
    """Gradients that nobody asks for are left out, the others keep their bits."""
    c = _case(40, 300, gate)
    rng = np.random.RandomState(7)
    x, rstd, rho = _stored(c)
    d = [rng.standard_normal(x.shape).astype(np.float32) for _ in range(2)]
    whole = _backward(c, gate, x, rstd, rho, *d)
    names = ("d_residual", "d_block", "d_gate", "d_post_weight", "d_pre_weight")
    for name in names:
        got = _backward(c, gate, x, rstd, rho, *d, leave_out=(name,))
        assert len(got) == len(whole) - 1 and all(np.array_equal(got[k], whole[k]) for k in got)
        got = _backward(c, gate, x, rstd, rho, *d, leave_out=[n for n in names if n != name])
        assert len(got) == 1 and all(np.array_equal(got[k], whole[k]) for k in got)


@pytest.mark.gpu
def test_no_rows():
    """Nothing to norm; the sums over no rows are zero."""
    c = _case(0, 12, "feature")
    _forward(c, "feature")
    e = np.zeros((0, 12), np.float32)
    got = _backward(c, "feature", e, np.zeros(0), np.zeros(0), e, e)
    assert not got["pre"].any() and not got["post"].any() and not got["gate"].any()
    got = _backward(_case(0, 12, block=False, post=False), "none", e, np.zeros(0), None, None, None)
    assert set(got) == {"residual", "pre"} and not got["pre"].any()


@pytest.mark.gpu
def test_rows_of_zeros_and_of_infinities():
    """A row of zeros is normalised to zeros; what is not finite stays in its row, and in the sums over rows."""
    c = _case(6, 200, "row")
    c["block"][1] = 0
    c["residual"][1] = 0
    c["residual"][3, 7], c["block"][4, 9] = np.inf, np.nan
    with np.errstate(all="ignore"):
        got, _ = _forward(c, "row")
    good = [0, 1, 2, 5]
    assert not got["out"][1].any() and np.all(np.isfinite(got["out"][good])) and np.all(np.isfinite(got["stream"][good]))
    assert np.isnan(got["out"][4]).all() and np.isnan(got["out"][3, 7])
    want, size = no.forward(c["residual"][good], c["block"][good], c["gate"][good], c["post"], c["pre"], c["a"], 1e-6)
    assert np.all(np.abs(got["out"][good] - want["out"]) <= 40 * HALF * size["out"])
    x, rstd, rho = [got[k] for k in ("stream", "stream_rstd", "block_rstd")]
    d = np.ones_like(x)
    back = _backward(c, "row", x, rstd, rho, d, d)
    assert np.all(np.isfinite(back["residual"][good])) and np.all(np.isfinite(back["block"][good])) and np.all(np.isfinite(back["gate"][good]))
    assert not np.all(np.isfinite(back["pre"]))


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "feature", "row", "full"])
def test_gradients_against_differences(gate):
    """The derivative along a direction by the kernel's gradients and by the kernel's own forward pass, either side.
    h = 1/64: the difference is off by h^2 / 6 of a third derivative of about the values' size, 4e-5, and by 2^-24 / h of
    a result's size from rounding, 4e-6, of the sizes' sum in all: 1e-3 of it is ample."""
    c = _case(11, 70, gate, seed=3)
    rng = np.random.RandomState(8)
    wo, ws = [rng.standard_normal(c["residual"].shape) for _ in range(2)]
    got, _ = _forward(c, gate)
    back = _backward(c, gate, got["stream"], got["stream_rstd"], got["block_rstd"], wo.astype(np.float32), ws.astype(np.float32))

    def value(shift):
        moved = dict(c)
        moved.update(shift)
        g, _ = _forward(moved, gate)
        return float((g["out"] * wo).sum() + (g["stream"] * ws).sum()), float(np.abs(g["out"] * wo).sum() + np.abs(g["stream"] * ws).sum())
    for name in ("residual", "block", "gate", "post", "pre"):
        if c[name] is None:
            continue
        v = rng.standard_normal(c[name].shape).astype(np.float32)
        h = 1.0 / 64
        up, size = value({name: c[name] + np.float32(h) * v})
        down, _ = value({name: c[name] - np.float32(h) * v})
        assert abs((up - down) / (2 * h) - float((back[name].reshape(v.shape).astype(np.float64) * v).sum())) <= 1e-3 * size, name


def test_the_oracles_gradients_against_autograd():
    import torch
    for gate in GATES:
        c = _case(5, 9, gate)
        t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in c.items() if isinstance(v, np.ndarray)}

        def rms(x):
            return x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)
        y = rms(t["block"]) * t["post"]
        s = c["a"] * t["residual"] + (y if c["gate"] is None else y * t["gate"])
        rng = np.random.RandomState(2)
        do, ds = [torch.tensor(rng.standard_normal((5, 9))) for _ in range(2)]
        ((rms(s) * t["pre"] * do).sum() + (s * ds).sum()).backward()
        f, _ = no.forward(c["residual"], c["block"], c["gate"], c["post"], c["pre"], c["a"], 1e-6)
        want, _ = no.backward(f["stream"], f["stream_rstd"], do.numpy(), ds.numpy(), c["block"], f["block_rstd"], c["gate"], c["post"], c["pre"], c["a"])
        for k, v in want.items():
            np.testing.assert_allclose(v, t[k].grad.numpy(), rtol=1e-10, atol=1e-10)


@pytest.mark.gpu
def test_recorded_and_replayed():
    """Forward and backward in one graph, replayed on other values."""
    import torch
    from ngraph_python_b200 import lib
    rows, F = 50, 768
    c = _case(rows, F, "feature")
    dev = {k: _vec(v) for k, v in c.items() if isinstance(v, np.ndarray)}
    rows_of = lambda: torch.zeros((rows, F), device="cuda")  # noqa: E731
    stream, out, d_out, d_res, d_block = [rows_of() for _ in range(5)]
    rstd, rho, d_pre, d_post, d_gate = [torch.zeros((n,), device="cuda") for n in (rows, rows, F, F, F)]
    a, d = lib.NormArgs(), lib.NormGrads()
    a.rows, a.features, a.gate_kind, a.residual_scale, a.eps = rows, F, 1, c["a"], 1e-6
    a.block_stride = a.residual_stride = a.stream_stride = a.out_stride = F
    a.block, a.residual, a.gate, a.post_weight, a.pre_weight = [dev[k].data_ptr() for k in ("block", "residual", "gate", "post", "pre")]
    a.stream, a.out, a.block_rstd, a.stream_rstd = [x.data_ptr() for x in (stream, out, rho, rstd)]
    d.d_out_stride = d.d_residual_stride = d.d_block_stride = F
    d.d_out, d.d_residual, d.d_block = d_out.data_ptr(), d_res.data_ptr(), d_block.data_ptr()
    d.d_pre_weight, d.d_post_weight, d.d_gate = d_pre.data_ptr(), d_post.data_ptr(), d_gate.data_ptr()
    nbytes = lib.norm_bprop_scratch_bytes(a)
    scratch = torch.empty((nbytes,), dtype=torch.uint8, device="cuda")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            st = torch.cuda.current_stream().cuda_stream
            lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), st))
            lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch.data_ptr(), nbytes, st))
        for seed in range(3):
            rng = np.random.RandomState(seed)
            c["block"] = rng.standard_normal((rows, F)).astype(np.float32)
            do = rng.standard_normal((rows, F)).astype(np.float32)
            dev["block"].copy_(torch.from_numpy(c["block"]))
            d_out.copy_(torch.from_numpy(do))
            graph.replay()
            side.synchronize()
            _check_forward(dict(stream=stream.cpu().numpy(), out=out.cpu().numpy(), stream_rstd=rstd.cpu().numpy()), c, F)
            got = dict(residual=d_res, block=d_block, pre=d_pre, post=d_post, gate=d_gate)
            _check_backward({k: v.cpu().numpy() for k, v in got.items()}, c, stream.cpu().numpy(), rstd.cpu().numpy(), rho.cpu().numpy(), do, None)


@pytest.mark.gpu
def test_large_offsets():
    """Rows that lie further than 2^31 values apart."""
    import torch
    from ngraph_python_b200 import lib
    F, stride = 64, 1 << 30
    x, y = [torch.empty((3 * stride + F,), device="cuda") for _ in range(2)]
    rows = torch.as_strided(x, (4, F), (stride, 1))
    rows.copy_(torch.randn(4, F))
    w = torch.ones((F,), device="cuda")
    a = lib.NormArgs()
    a.rows, a.features, a.residual_scale, a.eps = 4, F, 1.0, 1e-6
    a.residual, a.out, a.pre_weight, a.residual_stride, a.out_stride = x.data_ptr(), y.data_ptr(), w.data_ptr(), stride, stride
    lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), 0))
    got = torch.as_strided(y, (4, F), (stride, 1)).double()
    want = rows.double() / torch.sqrt((rows.double() ** 2).mean(1, keepdim=True) + 1e-6)
    assert float((got - want).abs().max()) <= 30 * HALF * float(want.abs().max())


def _whole():
    """Arguments that would be taken, and nothing behind them."""
    from ngraph_python_b200 import lib
    a, d = lib.NormArgs(), lib.NormGrads()
    a.rows, a.features, a.gate_kind, a.residual_scale, a.eps = 4, 8, 1, 0.5, 1e-6
    for k in ("block", "residual", "gate", "post_weight", "pre_weight", "stream", "out", "block_rstd", "stream_rstd"):
        setattr(a, k, 256)
    for k in ("block", "residual", "gate", "stream", "out"):
        setattr(a, k + "_stride", 8)
    for k in ("d_out", "d_stream", "d_residual", "d_block", "d_gate", "d_post_weight", "d_pre_weight"):
        setattr(d, k, 256)
    for k in ("d_out", "d_stream", "d_residual", "d_block", "d_gate"):
        setattr(d, k + "_stride", 8)
    return a, d


def test_refusals():
    from ngraph_python_b200 import lib
    raw = lib.raw()
    for kw in (dict(rows=-1), dict(features=0), dict(features=-4), dict(gate_kind=4), dict(gate_kind=0), dict(gate=None), dict(residual=None),
               dict(stream=None), dict(out=None), dict(pre_weight=None), dict(block=None), dict(block_stride=7), dict(residual_stride=-8),
               dict(stream_stride=4), dict(out_stride=0), dict(gate_kind=3, gate_stride=3),
               dict(block=None, gate=None, gate_kind=0, post_weight=None, stream=None),
               dict(block=None, gate=None, gate_kind=0, post_weight=None, stream=None, residual_scale=1.0, out=None, pre_weight=None)):
        a, _ = _whole()
        for k, v in kw.items():
            setattr(a, k, v)
        with pytest.raises(lib.B200Error, match="error -1"):
            lib.check(raw.b2_norm_fprop(ctypes.byref(a), 0))
    with pytest.raises(lib.B200Error, match="error -1"):
        lib.check(raw.b2_norm_fprop(None, 0))
    for kw, dkw in ((dict(rows=-1), {}), (dict(pre_weight=None), {}), ({}, dict(d_out=None)), (dict(pre_weight=None), dict(d_out=None)),
                    (dict(pre_weight=None), dict(d_out=None, d_pre_weight=None, d_stream=None)), (dict(stream_rstd=None), {}), (dict(block_rstd=None), {}),
                    (dict(stream=None), {}), (dict(gate=None, gate_kind=0), {}), (dict(post_weight=None), {}), ({}, dict(d_residual_stride=1)),
                    ({}, dict(d_block_stride=7)), ({}, dict(d_out_stride=0)), (dict(gate_kind=3), dict(d_gate_stride=1)), (dict(block_stride=2), {}),
                    (dict(block=None, gate=None, gate_kind=0, post_weight=None, residual_scale=1.0), {})):
        a, d = _whole()
        for k, v in kw.items():
            setattr(a, k, v)
        for k, v in dkw.items():
            setattr(d, k, v)
        with pytest.raises(lib.B200Error, match="error -1"):
            lib.check(raw.b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), 256, 1 << 24, 0))
    a, d = _whole()
    for scratch, nbytes in ((None, 1 << 24), (256, 8)):
        with pytest.raises(lib.B200Error, match="error -1"):
            lib.check(raw.b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch, nbytes, 0))


def _apart(**places):
    """The same with every tensor in a place of its own, but for those named."""
    a, d = _whole()
    names = [(a, k) for k in ("block", "residual", "gate", "post_weight", "pre_weight", "stream", "out", "block_rstd", "stream_rstd")] + \
        [(d, k) for k in ("d_out", "d_stream", "d_residual", "d_block", "d_gate", "d_post_weight", "d_pre_weight")]
    at = {k: (1 << 20) + 4096 * n for n, (_, k) in enumerate(names)}
    for x, k in names:
        setattr(x, k, at[places[k]] if k in places else at[k])
    return a, d


def test_results_in_the_place_of_operands_are_refused():
    from ngraph_python_b200 import lib

    def message(forward, a, d):
        with pytest.raises(lib.B200Error) as e:                  # (addresses of nothing: refused in any case)
            lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), 0) if forward else
                      lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), 256, 1 << 24, 0))
        return str(e.value)
    results, operands = ("out", "stream", "block_rstd", "stream_rstd"), ("block", "residual", "gate", "post_weight", "pre_weight")
    for r in results:
        for o in operands:
            assert ("place" in message(True, *_apart(**{r: o}))) == ((r, o) != ("stream", "residual"))
        for o in set(results) - {r}:
            assert "one place" in message(True, *_apart(**{r: o}))
    results = ("d_residual", "d_block", "d_gate", "d_post_weight", "d_pre_weight")
    for r in results:
        for o in ("d_out", "d_stream", "stream", "block", "gate", "post_weight", "pre_weight", "block_rstd", "stream_rstd"):
            assert ("place" in message(False, *_apart(**{r: o}))) == ((r, o) != ("d_residual", "d_stream"))
        for o in set(results) - {r}:
            assert "one place" in message(False, *_apart(**{r: o}))
    for forward, place in ((True, dict(stream="residual")), (False, dict(d_residual="d_stream"))):
        a, d = _apart(**place)
        assert "strides" not in message(forward, a, d)
        a.stream_stride, d.d_residual_stride = 12, 12
        assert "other strides" in message(forward, a, d)
        a.rows = 1
        assert "strides" not in message(forward, a, d)


@pytest.mark.gpu
def test_host_memory_is_refused():
    import torch
    from ngraph_python_b200 import lib
    rows, F = 3, 8
    host = np.ones((rows, F), np.float32)
    c = _case(rows, F, "full")
    _, (a, mem, vecs) = _forward(c, "full")
    for name in ("residual", "block", "gate", "stream", "out"):
        held = getattr(a, name)
        setattr(a, name, host.ctypes.data)
        with pytest.raises(lib.B200Error, match="memory"):
            lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), 0))
        setattr(a, name, held)
    t = {k: torch.ones((rows, F), device="cuda") for k in ("d_out", "d_stream", "d_residual", "d_block", "d_gate")}
    d = lib.NormGrads()
    for k, v in t.items():
        setattr(d, k, v.data_ptr())
        setattr(d, k + "_stride", F)
    nbytes = lib.norm_bprop_scratch_bytes(a)
    scratch = torch.zeros((max(nbytes, 256),), dtype=torch.uint8, device="cuda")
    for name in t:
        held = getattr(d, name)
        setattr(d, name, host.ctypes.data)
        with pytest.raises(lib.B200Error, match="memory"):
            lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch.data_ptr(), scratch.numel(), 0))
        setattr(d, name, held)
    lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch.data_ptr(), scratch.numel(), 0))
    torch.cuda.synchronize()
    assert (host == 1).all()


def test_sums_over_no_rows_in_one_place_are_refused():
    from ngraph_python_b200 import lib
    for pair in (("d_pre_weight", "d_post_weight"), ("d_gate", "d_pre_weight"), ("d_gate", "d_post_weight")):
        a, d = _apart(**{pair[0]: pair[1]})
        a.rows = 0
        with pytest.raises(lib.B200Error, match="one place"):
            lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), 256, 1 << 24, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 3])
def test_vectors_in_host_memory_are_refused(rows):
    """The reciprocal deviations, the weights, and sums over rows, which are written for no rows too."""
    import torch
    from ngraph_python_b200 import lib
    F = 8
    host = np.ones((64,), np.float32)
    t = {k: torch.ones((4, F), device="cuda") for k in ("block", "residual", "gate", "post_weight", "pre_weight", "stream", "out", "block_rstd", "stream_rstd",
                                                        "d_out", "d_stream", "d_residual", "d_block", "d_gate", "d_post_weight", "d_pre_weight")}
    a, d = _whole()
    a.rows = rows
    for x in (a, d):
        for k, v in t.items():
            if hasattr(x, k):
                setattr(x, k, v.data_ptr())
    scratch = torch.zeros((lib.norm_bprop_scratch_bytes(a) + 256,), dtype=torch.uint8, device="cuda")
    forward = lambda: lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), 0))  # noqa: E731
    backward = lambda: lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch.data_ptr(), scratch.numel(), 0))  # noqa: E731

    def refused(call, x, name):
        held = getattr(x, name)
        setattr(x, name, host.ctypes.data)
        with pytest.raises(lib.B200Error, match="memory"):
            call()
        setattr(x, name, held)
    for name in ("d_post_weight", "d_pre_weight", "d_gate"):
        refused(backward, d, name)
    if rows:
        for name in ("block_rstd", "stream_rstd", "post_weight", "pre_weight"):
            refused(forward, a, name)
            refused(backward, a, name)
    forward()
    backward()
    torch.cuda.synchronize()
    assert (host == 1).all()


def test_addresses_between_two_values_are_refused():
    from ngraph_python_b200 import lib
    for rows in (0, 4):
        for forward in (True, False):
            a, d = _apart()
            for x in (a, d) if not forward else (a,):
                for k in [k for k, t in x._fields_ if t is ctypes.c_void_p and k != "status"]:
                    for by in (1, 2, 3, 4):
                        a, d = _apart()
                        a.rows = rows
                        y = a if type(x) is type(a) else d
                        setattr(y, k, getattr(y, k) + by)
                        call = lambda: lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), 0) if forward else  # noqa: E731
                                                 lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), 256, 1 << 24, 0))
                        if by % 4:
                            with pytest.raises(lib.B200Error, match="between two addresses"):
                                call()
                        elif rows or not forward:
                            with pytest.raises(lib.B200Error) as e:      # (addresses of nothing: refused in any case)
                                call()
                            assert "between" not in str(e.value)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["feature", "row", "full"])
@pytest.mark.parametrize("rows,F", [(5, 64), (700, 37), (40, 2048), (6, 1001)])
def test_operands_in_page_locked_memory(rows, F, gate):
    """All of them at once, and the rows of one at a time."""
    import torch
    from ngraph_python_b200 import lib
    rng = np.random.RandomState(4)
    c = _case(rows, F, gate)
    x, rstd, rho = _stored(c)
    d_out, d_stream = [rng.standard_normal((rows, F)).astype(np.float32) for _ in range(2)]
    host = dict(residual=c["residual"], block=c["block"], gate=c["gate"], post_weight=c["post"], pre_weight=c["pre"], stream=x, stream_rstd=rstd,
                block_rstd=rho, d_out=d_out, d_stream=d_stream)
    host = {k: torch.from_numpy(np.ascontiguousarray(v, dtype=np.float32)).pin_memory() for k, v in host.items()}
    device = {k: v.cuda() for k, v in host.items()}
    for locked in (tuple(host), ("residual",), ("block",), ("gate",), ("stream",), ("d_out",), ("d_stream",)):
        at = {k: (host if k in locked else device)[k].data_ptr() for k in host}
        a = lib.NormArgs(rows=rows, features=F, gate_kind=GATES[gate], residual_scale=c["a"], eps=1e-6)
        for k in ("block", "residual", "gate", "stream", "out"):
            setattr(a, k + "_stride", F)
        for k in ("block", "residual", "gate", "post_weight", "pre_weight"):
            setattr(a, k, at[k])
        got = {k: torch.zeros(s, device="cuda") for k, s in (("stream", (rows, F)), ("out", (rows, F)), ("stream_rstd", (rows,)), ("block_rstd", (rows,)))}
        for k, v in got.items():
            setattr(a, k, v.data_ptr())
        lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), 0))
        torch.cuda.synchronize()
        _check_forward({k: v.cpu().numpy() for k, v in got.items()}, c, F)
        for k in ("stream", "stream_rstd", "block_rstd"):
            setattr(a, k, at[k])
        d = lib.NormGrads(d_out=at["d_out"], d_stream=at["d_stream"])
        got = {k: torch.zeros(s, device="cuda") for k, s in (("d_residual", (rows, F)), ("d_block", (rows, F)), ("d_gate", c["gate"].shape),
                                                            ("d_post_weight", (F,)), ("d_pre_weight", (F,)))}
        for k in ("d_out", "d_stream", "d_residual", "d_block", "d_gate"):
            setattr(d, k + "_stride", F)
        for k, v in got.items():
            setattr(d, k, v.data_ptr())
        nbytes = lib.norm_bprop_scratch_bytes(a)
        scratch = torch.full((nbytes,), 0xA5, dtype=torch.uint8, device="cuda")
        lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch.data_ptr(), nbytes, 0))
        torch.cuda.synchronize()
        names = dict(d_residual="residual", d_block="block", d_gate="gate", d_post_weight="post", d_pre_weight="pre")
        _check_backward({names[k]: v.cpu().numpy() for k, v in got.items()}, c, x, rstd, rho, d_out, d_stream)


def _held(base, rows, width, stride):
    return set(base // 4 + i * stride + k for i in range(rows) for k in range(width))


@pytest.mark.parametrize("forward", [True, False])
def test_results_that_overlap_are_refused(forward):
    """Two tensors at a time near one another, with strides of their own: refused where they share a value and one is
    written, and not where their rows lie side by side."""
    from ngraph_python_b200 import lib
    rng = np.random.RandomState(3 + forward)
    rowed = ("block", "residual", "gate", "stream", "out") if forward else ("block", "gate", "stream", "d_out", "d_stream", "d_residual", "d_block", "d_gate")
    vectors = ("post_weight", "pre_weight", "block_rstd", "stream_rstd") + (() if forward else ("d_post_weight", "d_pre_weight"))
    results = ("stream", "out", "block_rstd", "stream_rstd") if forward else ("d_residual", "d_block", "d_gate", "d_post_weight", "d_pre_weight")
    seen = {True: 0, False: 0}
    for _ in range(4000):
        a, d = _apart()
        a.gate_kind, a.features, a.rows = 3, int(rng.randint(1, 7)), int(rng.randint(1, 6))
        F, R = a.features, a.rows
        of = lambda k: a if hasattr(a, k) else d  # noqa: E731
        strides = {k: int(F + rng.choice([0, 0, F, 2 * F, rng.randint(0, 9)])) for k in rowed}
        if rng.rand() < 0.5:
            strides = dict.fromkeys(rowed, strides[rowed[0]])
        for k in rowed:
            setattr(of(k), k + "_stride", strides[k])
        x, y = [str(k) for k in rng.choice(rowed + vectors, 2, replace=False)]
        if {x, y} in ({"residual", "stream"}, {"d_residual", "d_stream"}):
            continue                                # (these may share memory; the strides then have to agree)
        setattr(of(y), y, getattr(of(x), x) + 4 * int(rng.randint(-30, 31)))
        held = [_held(getattr(of(k), k), R, F, strides[k]) if k in rowed else _held(getattr(of(k), k), 1, R if k.endswith("rstd") else F, 0) for k in (x, y)]
        wrong = bool(held[0] & held[1]) and (x in results or y in results)
        with pytest.raises(lib.B200Error) as e:      # (addresses of nothing: refused in any case)
            lib.check(lib.raw().b2_norm_fprop(ctypes.byref(a), 0) if forward else
                      lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), 256, 1 << 24, 0))
        text = str(e.value)
        assert any(t in text for t in ("overlaps an operand", "norm overlap", "place")) == wrong, (x, y, text)
        seen[wrong] += 1
    assert min(seen.values()) > 500


def test_a_scratch_that_overlaps_is_refused():
    from ngraph_python_b200 import lib
    for rows in (0, 4):
        a, d = _apart()
        a.rows = rows
        need = lib.norm_bprop_scratch_bytes(a)
        for k in ("d_post_weight", "d_pre_weight") + (("stream", "d_out", "d_residual", "block_rstd") if rows else ()):
            at = getattr(a if hasattr(a, k) else d, k)
            for scratch, overlaps in ((at - need + 8, True), (at, True), (at + 4, True), (at - need, False)):
                with pytest.raises(lib.B200Error) as e:      # (addresses of nothing: refused in any case)
                    lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch, need, 0))
                assert any(t in str(e.value) for t in ("overlap", "place")) == overlaps


def test_a_status_between_addresses_is_refused():
    from ngraph_python_b200 import lib
    a, d = _apart()
    d.status = 258
    with pytest.raises(lib.B200Error, match="status lies between"):
        lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), 256, 1 << 24, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,F", [(3, 8), (700, 37), (900, 1001), (200, 8192)])
def test_the_status_stays_as_it_is_where_no_wait_runs_out(rows, F):
    import torch
    from ngraph_python_b200 import lib
    c = _case(rows, F, "row")
    rng = np.random.RandomState(5)
    x, rstd, rho = _stored(c)
    rows_of = dict(block=c["block"], stream=x, d_out=rng.standard_normal((rows, F)), d_stream=rng.standard_normal((rows, F)))
    t = {k: _vec(v) for k, v in dict(rows_of, gate=c["gate"], post_weight=c["post"], pre_weight=c["pre"], stream_rstd=rstd, block_rstd=rho).items()}
    grads = {k: torch.zeros(s, device="cuda") for k, s in (("d_residual", (rows, F)), ("d_block", (rows, F)), ("d_gate", (rows,)), ("d_post_weight", (F,)),
                                                          ("d_pre_weight", (F,)))}
    status = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    a, d = lib.NormArgs(rows=rows, features=F, gate_kind=2, residual_scale=c["a"], eps=1e-6), lib.NormGrads(status=status.data_ptr())
    for y, held in ((a, t), (d, dict(t, **grads))):
        for k, v in held.items():
            if hasattr(y, k):
                setattr(y, k, v.data_ptr())
            if hasattr(y, k + "_stride"):
                setattr(y, k + "_stride", F)
    scratch = torch.zeros((lib.norm_bprop_scratch_bytes(a),), dtype=torch.uint8, device="cuda")
    call = lambda: lib.check(lib.raw().b2_norm_bprop(ctypes.byref(a), ctypes.byref(d), scratch.data_ptr(), scratch.numel(), 0))  # noqa: E731
    call()
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0]
    names = dict(d_residual="residual", d_block="block", d_gate="gate", d_post_weight="post", d_pre_weight="pre")
    _check_backward({names[k]: v.cpu().numpy() for k, v in grads.items()}, c, x, rstd, rho, rows_of["d_out"].astype(np.float32),
                    rows_of["d_stream"].astype(np.float32))
    d.status = status.cpu().data_ptr()
    with pytest.raises(lib.B200Error, match="memory"):
        call()
