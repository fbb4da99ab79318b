"""The optimizer step of orthogonalised updates through the C ABI, against 64 bits."""
import ctypes

import numpy as np
import pytest

from oracle import muon_oracle as mo

HALF = 2.0 ** -24
STEP = dict(lr=0.02, momentum=0.95, eps=1e-7, weight_decay=0.1, a=mo.A, b=mo.B, c=mo.C, steps=5, nesterov=1)


def _data(r, c, seed=0, kind="gauss"):
    rng = np.random.RandomState(seed + 7 * r + c)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    grad, mean = f(r, c), f(r, c) * np.float32(0.5)
    if kind == "few":                   # a few directions outweigh the others by far
        grad = (1e-3 * grad + f(r, 2) @ f(2, c)).astype(np.float32)
        mean = (1e-3 * mean).astype(np.float32)
    return dict(param=f(r, c) * np.float32(0.05), grad=grad, mean=mean)


class _Step(object):
    """Matrices on the device, each in a sea of marks, with their plan and scratch."""
    MARK = -77.0

    def __init__(self, data, offset=0, decay=None, scale=None, hyper=None, lr=None, grad_scale=None, step=None):
        import torch
        from ngraph_python_b200 import lib
        self.lib, self.torch = lib, torch
        self.shapes = [d["param"].shape for d in data]
        self.all = [{k: torch.full((v.size + offset + 4,), self.MARK, device="cuda") for k, v in d.items()} for d in data]
        self.offset = offset
        for on, d in zip(self.all, data):
            for k, v in d.items():
                on[k][offset:offset + v.size] = torch.from_numpy(v.ravel()).cuda()
        m = (lib.MuonMatrix * len(data))()
        for i, (x, (r, c), on) in enumerate(zip(m, self.shapes, self.all)):
            x.param, x.grad, x.mean = [on[k].data_ptr() + 4 * offset for k in ("param", "grad", "mean")]
            x.rows, x.cols = r, c
            x.decay, x.scale = 1.0 if decay is None else decay[i], 1.0 if scale is None else scale[i]
        self.sizes = lib.muon_plan_sizes(m)
        self.plan = torch.empty((self.sizes.plan_bytes + 64,), dtype=torch.uint8, device="cuda")
        lib.muon_plan(m, self.plan.data_ptr(), self.sizes.plan_bytes, torch.cuda.current_stream().cuda_stream)
        self.scratch = torch.full((self.sizes.scratch_bytes + 64,), 255, dtype=torch.uint8, device="cuda")
        self.hyper = lib.MuonHyper(**dict(STEP, **(hyper or {})))
        number = lambda v: None if v is None else torch.full((1,), float(v), device="cuda")  # noqa: E731
        self.numbers = [number(v) for v in (lr, grad_scale, step)]
        self.status = torch.zeros((1,), dtype=torch.int32, device="cuda")

    def __call__(self, stream=None):
        at = [None if v is None else v.data_ptr() for v in self.numbers]
        self.lib.check(self.lib.raw().b2_muon_step(self.plan.data_ptr(), ctypes.byref(self.sizes), ctypes.byref(self.hyper), *at,
                                                   self.scratch.data_ptr(), self.sizes.scratch_bytes, self.status.data_ptr(), stream))

    def get(self):
        self.torch.cuda.synchronize()
        assert int(self.status[0]) == 0
        o, found = self.offset, []
        for (r, c), on in zip(self.shapes, self.all):
            assert all(bool((v[:o] == self.MARK).all()) and bool((v[o + r * c:] == self.MARK).all()) for v in on.values())
            found.append({k: v[o:o + r * c].cpu().numpy().reshape(r, c) for k, v in on.items()})
        assert self.scratch[self.sizes.scratch_bytes:].eq(255).all()
        return found


def _check(got, d, scale=1.0, decay=1.0, grad_scale=1.0, mu=0.95, nesterov=True, hyper=None):
    """The mean to the rounding of its two products and their sum; the param to where the iteration may be carried, and the
    rounding of its own two products and difference."""
    h = dict(STEP, **(hyper or {}))
    x, mean = mo.update(d["grad"], d["mean"], mu, h["eps"], nesterov, grad_scale)
    size = mu * np.abs(d["mean"]) + (1 - mu) * np.abs(grad_scale * d["grad"])
    assert np.all(np.abs(got["mean"] - mean) <= 5 * HALF * size)
    poly = {k: h[k] for k in ("steps", "a", "b", "c")}
    want, _ = mo.orthogonal(x, **poly)
    move = h["lr"] * scale
    want = d["param"] * (1 - h["lr"] * h["weight_decay"] * decay) - move * want
    # (the operand itself is off by the roundings of u, of its norm and of their quotient: 8 units)
    own = mo.reach(x, **poly) + 8 * HALF * np.sqrt(np.sum(x * x)) * 4 ** h["steps"]
    off = np.sqrt(np.sum((got["param"] - want) ** 2))
    rounding = 4 * HALF * np.sqrt(np.sum(d["param"].astype(np.float64) ** 2) + np.sum(want ** 2))
    assert off <= abs(move) * own + rounding, (off, abs(move) * own, rounding)
    return off / max(abs(move), 1e-30)


SHAPES = [(1, 1), (1, 640), (129, 1), (2, 3), (64, 64), (63, 65), (128, 128), (77, 77), (65, 300), (300, 65), (301, 1001), (1001, 301), (130, 127), (16, 4096),
          (640, 192), (257, 513), (513, 257), (192, 640), (64, 512), (64, 768), (64, 769), (768, 33), (520, 64), (65, 256), (128, 256), (128, 257), (256, 100), (2, 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("r,c", SHAPES)
@pytest.mark.parametrize("kind,offset", [("gauss", 0), ("few", 1)])
def test_one_matrix(r, c, kind, offset):
    d = _data(r, c, kind=kind)
    s = _Step([d], offset)
    s()
    _check(s.get()[0], d)


@pytest.mark.gpu
def test_the_orthogonalised_matrix_itself():
    """Onto a param of zeros at a rate of one: the update alone, whose singular values lie where the polynomial takes them."""
    for r, c in ((96, 160), (200, 70), (384, 384)):
        d = _data(r, c)
        d["param"][:] = 0
        s = _Step([d], hyper=dict(lr=1.0, weight_decay=0.0))
        s()
        got = s.get()[0]
        off = _check(got, d, hyper=dict(lr=1.0, weight_decay=0.0))
        x = mo.update(d["grad"], d["mean"])[0]
        want = mo.orthogonal(x)[0]
        # as exact as products in fp32 are: against the same in numpy's 32 bits, four times as far at most
        y = (x.T if r > c else x).astype(np.float32)
        for _ in range(5):
            a = y @ y.T
            y = np.float32(mo.A) * y + (np.float32(mo.B) * a + np.float32(mo.C) * (a @ a)) @ y
        plain = np.sqrt(np.sum(((y.T if r > c else y) - want) ** 2))
        assert off <= 4 * plain + 8 * HALF * np.sqrt(np.sum(want ** 2)), (off, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 3])
def test_many_matrices_and_rates(offset):
    """Sizes next to one another, empty ones among them; rates and scales on the device, three steps; the number of steps."""
    shapes = [(64, 192), (0, 5), (77, 77), (301, 100), (1, 7), (5, 0), (129, 1), (200, 333), (64, 64), (512, 40)]
    data = [_data(r, c, seed=i) for i, (r, c) in enumerate(shapes)]
    decay, scale = [float(i % 2) for i in range(10)], [1.0 + 0.25 * i for i in range(10)]
    for nesterov, mu in ((1, 0.95), (0, 0.5), (1, 0.0)):
        s = _Step(data, offset, decay, scale, hyper=dict(nesterov=nesterov, momentum=mu, lr=9.0), lr=0.5, grad_scale=0.25, step=41)
        before = data
        for n in range(3):
            s()
            found = s.get()
            for d, got, de, sc in zip(before, found, decay, scale):
                _check(got, d, sc, de, 0.25, mu, nesterov, hyper=dict(lr=0.5))
                assert np.array_equal(got["grad"], d["grad"])
            before = found
            assert float(s.numbers[2][0]) == 42.0 + n


@pytest.mark.gpu
@pytest.mark.parametrize("poly", [dict(a=1.5, b=-0.5, c=0.0, steps=8), dict(a=2.0, b=-1.5, c=0.5, steps=1), dict(a=3.4445, b=-4.775, c=2.0315, steps=2),
                                  dict(a=1.875, b=-1.25, c=0.375, steps=12)])
def test_other_polynomials(poly):
    for r, c in ((70, 130), (130, 70)):
        d = _data(r, c)
        s = _Step([d], hyper=poly)
        s()
        _check(s.get()[0], d, hyper=poly)


@pytest.mark.gpu
def test_the_same_bits_in_every_run_and_in_a_recording():
    data = [_data(r, c) for r, c in ((320, 500), (64, 64), (500, 320), (31, 77))]
    runs = []
    for k in range(3):
        s = _Step(data)
        if k == 2:
            st, graph = s.torch.cuda.Stream(), s.torch.cuda.CUDAGraph()
            with s.torch.cuda.graph(graph, stream=st):
                s(st.cuda_stream)
            graph.replay()
            graph.replay()
        else:
            s.scratch[:s.sizes.scratch_bytes].random_(0, 255)
            s()
            s()
        runs.append(s.get())
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert all(np.array_equal(a[k], b[k]) for k in a)


@pytest.mark.gpu
def test_two_streams_at_once():
    torch = pytest.importorskip("torch")
    data = [[_data(r, c, seed=k) for r, c in ((256, 640), (640, 256), (77, 33))] for k in range(2)]
    alone = []
    for d in data:
        s = _Step(d)
        s()
        alone.append(s.get())
    steps, streams = [_Step(d) for d in data], [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    for s, st in zip(steps, streams):
        s(st.cuda_stream)
    for s, want in zip(steps, alone):
        for a, b in zip(s.get(), want):
            assert all(np.array_equal(a[k], b[k]) for k in a)


@pytest.mark.gpu
def test_zeros_and_values_that_are_not_finite():
    """Nothing to orthogonalise: the param decays.  An infinity or NaN spoils its own matrix alone; large and small gradients do not."""
    shapes = [(70, 90), (70, 90), (70, 90), (70, 90), (90, 70), (70, 90)]
    data = [_data(r, c, seed=i) for i, (r, c) in enumerate(shapes)]
    data[0]["grad"][:] = 0
    data[0]["mean"][:] = 0
    data[1]["grad"][3, 5] = np.inf
    data[2]["grad"][69, 89] = np.nan
    data[3]["grad"] *= np.float32(1e25)
    data[3]["mean"] *= np.float32(1e25)
    data[4]["grad"] *= np.float32(1e-30)
    data[4]["mean"] *= np.float32(1e-30)
    s = _Step(data, hyper=dict(eps=1e-37))
    s()
    got = s.get()
    keep = data[0]["param"] * (1 - 0.02 * 0.1)
    assert np.all(np.abs(got[0]["param"] - keep) <= 2 * HALF * np.abs(keep)) and not got[0]["mean"].any()
    assert np.isnan(got[1]["param"]).all() and np.isnan(got[2]["param"]).all()
    for i in (3, 4, 5):
        _check(got[i], data[i], hyper=dict(eps=1e-37))


@pytest.mark.gpu
def test_a_matrix_of_one_entry_and_one_direction():
    """The largest values that an operand can have: all of the norm in one entry, and a matrix of rank one."""
    for r, c in ((64, 64), (130, 70), (70, 200)):
        one, flat = _data(r, c), _data(r, c)
        for k in ("grad", "mean"):
            one[k][:] = 0
            one[k][r // 2, c // 3] = 5
            flat[k][:] = 1
        s = _Step([one, flat])
        s()
        got = s.get()
        _check(got[0], one)
        _check(got[1], flat)


@pytest.mark.gpu
def test_sizes_of_another_plan_and_no_matrices():
    data = [_data(40, 50), _data(64, 65)]
    s, other = _Step(data), _Step(data[:1])
    sizes, s.sizes = s.sizes, other.sizes
    s()
    s.torch.cuda.synchronize()
    s.sizes = sizes
    for got, d in zip(s.get(), data):
        assert all(np.array_equal(got[k], d[k]) for k in d)
    none = _Step([], step=3)
    none()
    assert none.get() == [] and float(none.numbers[2][0]) == 4.0


@pytest.mark.gpu
def test_gradients_that_are_shared_or_in_page_locked_memory():
    import torch
    from ngraph_python_b200 import lib
    d = _data(96, 130)
    s = _Step([d, d])
    pinned = torch.from_numpy(d["grad"].copy()).pin_memory()
    m = (lib.MuonMatrix * 2)()
    for x, on in zip(m, s.all):
        x.param, x.grad, x.mean, x.rows, x.cols, x.decay, x.scale = on["param"].data_ptr(), pinned.data_ptr(), on["mean"].data_ptr(), 96, 130, 1.0, 1.0
    lib.muon_plan(m, s.plan.data_ptr(), s.sizes.plan_bytes, torch.cuda.current_stream().cuda_stream)
    s()
    a, b = s.get()
    _check(a, d)
    assert np.array_equal(a["param"], b["param"])
    host = torch.zeros((96 * 130,)).pin_memory()
    m[0].param = host.data_ptr()
    with pytest.raises(lib.B200Error, match="not device memory"):
        lib.muon_plan(m, s.plan.data_ptr(), s.sizes.plan_bytes, 0)


@pytest.mark.gpu
def test_a_plan_is_not_made_in_a_recording():
    import torch
    s = _Step([_data(8, 8)])
    m = (s.lib.MuonMatrix * 1)()
    x = m[0]
    x.param, x.grad, x.mean, x.rows, x.cols = [s.all[0][k].data_ptr() for k in ("param", "grad", "mean")] + [8, 8]
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        with pytest.raises(s.lib.B200Error, match="captured"):
            s.lib.muon_plan(m, s.plan.data_ptr(), s.sizes.plan_bytes, st.cuda_stream)
        s(st.cuda_stream)


def test_refusals():
    from ngraph_python_b200 import lib

    def matrices(*changes):
        m = (lib.MuonMatrix * 2)()
        for i, x in enumerate(m):
            x.param, x.grad, x.mean, x.rows, x.cols, x.decay, x.scale = (1 << 20) + (i << 24), (2 << 20) + (i << 24), (3 << 20) + (i << 24), 8, 16, 1.0, 1.0
        for k, v in changes:
            setattr(m[0], k, v)
        return m

    for bad, text in ((("param", None), "missing address"), (("grad", None), "missing address"), (("mean", None), "missing address"), (("rows", -1), "sides"),
                      (("cols", -1), "sides"), (("rows", (1 << 20) + 1), "sides"), (("decay", float("nan")), "decay"), (("scale", float("inf")), "decay"),
                      (("param", (1 << 20) + 2), "between two addresses")):
        with pytest.raises(lib.B200Error, match=text):
            lib.muon_plan_sizes(matrices(bad))
    with pytest.raises(lib.B200Error, match="sides"):
        lib.muon_plan_sizes(matrices(("rows", 40000), ("cols", 40000)))
    sizes = lib.muon_plan_sizes(matrices())
    plan = lambda m, at=1 << 33, n=sizes.plan_bytes: lib.muon_plan(m, at, n)  # noqa: E731
    for m, text in ((matrices(("param", 3 << 20)), "overlap"), (matrices(("mean", (1 << 20) + 64)), "overlap"), (matrices(("param", (1 << 20) + (1 << 24))), "overlap"),
                    (matrices(("grad", (1 << 20) + 508)), "gradient 0 overlaps"), (matrices(("grad", 3 << 20)), "gradient 0 overlaps"),
                    (matrices(("param", (1 << 33) + 64)), "in its memory"), (matrices(("grad", 1 << 33)), "gradient 0 overlaps")):
        with pytest.raises(lib.B200Error, match=text):
            plan(m)
    with pytest.raises(lib.B200Error, match="the plan needs"):
        plan(matrices(), n=sizes.plan_bytes - 1)
    with pytest.raises(lib.B200Error, match="the plan needs"):
        plan(matrices(), at=None)

    def step(text, hyper=None, lr=None, grad_scale=None, count=None, scratch=1 << 34, nbytes=sizes.scratch_bytes, at=1 << 33, s=sizes, status=None):
        h = lib.MuonHyper(**dict(STEP, **(hyper or {})))
        rc = lib.raw().b2_muon_step(at, None if s is None else ctypes.byref(s), ctypes.byref(h), lr, grad_scale, count, scratch, nbytes, status, None)
        assert rc == -1 and text in lib.raw().b2_last_error().decode(), lib.raw().b2_last_error()
    for bad in (dict(lr=float("nan")), dict(momentum=1.0), dict(momentum=-0.1), dict(eps=-1.0), dict(weight_decay=float("inf")), dict(steps=0), dict(steps=33),
                dict(a=float("nan")), dict(c=float("inf"))):
        step("bad", bad)
    step("bad argument", at=None)
    step("bad argument", s=None)
    step("scratch", scratch=None)
    step("scratch", nbytes=sizes.scratch_bytes - 1)
    step("lies in the scratch", scratch=(1 << 33) + 64)
    for which in ("lr", "grad_scale", "count", "status"):
        step("between two addresses", **{which: (1 << 35) + 2})


def test_the_oracle_takes_singular_values_to_one():
    rng = np.random.RandomState(0)
    x = rng.standard_normal((20, 30))
    x /= np.sqrt(np.sum(x * x))
    y, _ = mo.orthogonal(x)
    s = np.linalg.svd(y, compute_uv=False)
    assert np.all(s > 0.6) and np.all(s < 1.3)
    u, t, v = np.linalg.svd(x, full_matrices=False)
    for _ in range(5):
        t = mo.A * t + mo.B * t ** 3 + mo.C * t ** 5
    assert np.allclose(y, (u * t) @ v, atol=1e-12)
