"""An AdamW step over many tensors, through the C ABI: bit for bit what numpy computes with every fp32 operation
rounded by itself, with moments in 32 and in 8 bits."""
import ctypes

import numpy as np
import pytest

from oracle import adamw_oracle as ao

HYPER = (3e-4, 0.9, 0.999, 1e-8, 0.1)


class _Model(object):
    """Tensors on the device and the same for the oracle."""

    def __init__(self, sizes, bits, seed=0, offset=0, before=0, decays=None, zero=False):
        import torch
        from ngraph_python_b200 import lib
        rng = np.random.RandomState(seed)
        self.bits, self.t, self.seed = bits, before, 1234567 + seed
        self.host, self.dev, self.grads = [], [], []
        self.decays = decays or [float(k % 2) for k in range(len(sizes))]
        self.counters = [int(rng.randint(0, 2 ** 32, dtype=np.uint64)) for _ in sizes]
        tensors = (lib.AdamwTensor * len(sizes))()

        def device(a, off):
            t = torch.zeros((a.size + off + 8,), dtype=torch.from_numpy(a[:0]).dtype, device="cuda")
            t[off:off + a.size] = torch.from_numpy(a)
            return t[off:off + a.size]
        for k, n in enumerate(sizes):
            p = rng.standard_normal(n).astype(np.float32)
            m = np.zeros(n, np.float32) if zero else (rng.standard_normal(n) * 1e-3).astype(np.float32)
            r = np.zeros(n, np.float32) if zero else np.abs(rng.standard_normal(n) * 10.0 ** rng.uniform(-6, -1, n)).astype(np.float32)
            if bits == 32:
                state = (m, r * r)
            else:
                codes, scales = [], []
                for x in (m, r):
                    blocks = -(-n // 256)
                    pad = np.zeros(blocks * 256, np.float32)
                    pad[:n] = x
                    top = np.abs(pad).reshape(-1, 256).max(1) if n else np.zeros(0, np.float32)
                    scales.append((top / np.float32(448)).astype(np.float32))
                    c = rng.randint(0, 127, n).astype(np.uint8) if not zero else np.zeros(n, np.uint8)
                    codes.append(c)
                codes[0] = codes[0] | (rng.randint(0, 2, n).astype(np.uint8) << 7) if not zero else codes[0]
                state = (codes[0], codes[1], scales[0], scales[1])
            g = (rng.standard_normal(n) * 1e-2).astype(np.float32)
            self.host.append([p, state])
            self.dev.append([device(p, offset), [device(s, offset) for s in state]])
            self.grads.append([g, device(g, offset)])
            x = tensors[k]
            x.param, x.grad, x.n = self.dev[k][0].data_ptr(), self.grads[k][1].data_ptr(), n
            x.m, x.v = [s.data_ptr() for s in self.dev[k][1][:2]]
            if bits == 8:
                x.m_scales, x.v_scales = [s.data_ptr() for s in self.dev[k][1][2:]]
            x.decay, x.counter = self.decays[k], self.counters[k]
        self.tensors = tensors
        nbytes, self.chunks = lib.adamw_plan_bytes(tensors, bits)
        self.plan = torch.empty((nbytes,), dtype=torch.uint8, device="cuda")
        lib.adamw_plan(tensors, bits, self.plan.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
        self.step_dev = torch.full((1,), float(before), device="cuda")

    def new_gradients(self, seed):
        import torch
        rng = np.random.RandomState(seed)
        for g in self.grads:
            g[0] = (rng.standard_normal(g[0].size) * 10.0 ** rng.uniform(-4, 0)).astype(np.float32)
            g[1].copy_(torch.from_numpy(g[0]))

    def launch(self, hyper=HYPER, lr=None, scale=None, stream=None):
        import torch
        from ngraph_python_b200 import lib
        h = lib.AdamwHyper(*hyper)
        at = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        lib.check(lib.raw().b2_adamw_step(self.plan.data_ptr(), self.chunks, self.bits, ctypes.byref(h), at(lr), at(scale), self.step_dev.data_ptr(),
                                          self.seed, torch.cuda.current_stream().cuda_stream if stream is None else stream))

    def expect(self, hyper=HYPER, scale=1.0):
        self.t += 1
        for k, (p, state) in enumerate(self.host):
            if p.size:
                self.host[k] = list(ao.step(p, self.grads[k][0], state, self.t, hyper, self.decays[k], scale, self.seed, self.counters[k]))

    def check(self):
        import torch
        torch.cuda.synchronize()
        assert float(self.step_dev) == self.t
        for (p, state), (dp, dstate) in zip(self.host, self.dev):
            assert np.array_equal(dp.cpu().numpy(), p)
            for s, d in zip(state, dstate):
                assert np.array_equal(d.cpu().numpy(), s)


SIZES = [[1], [2048], [7, 0, 255, 256, 257, 2047, 2049, 3], [100003, 1, 4096, 640], [16] * 700]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("offset", [0, 1])
def test_steps(bits, sizes, offset):
    m = _Model(sizes, bits, offset=offset, before=6)
    for k in range(3):
        m.new_gradients(k)
        m.launch()
        m.expect()
        m.check()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
def test_nothing_beside_the_tensors_is_touched(bits, offset):
    """Tensors in the midst of marked memory, whose lengths end blocks, words and chunks early."""
    import torch
    m = _Model([5, 255, 2051, 1], bits, offset=offset, before=4)
    around = []
    for p, state in m.dev:
        for t in [p] + list(state):
            whole = torch.as_strided(t, (offset + t.numel() + 8,), (1,), t.storage_offset() - offset)
            whole[:offset], whole[offset + t.numel():] = 77, 77
            around.append((whole, t.numel()))
    m.launch()
    m.expect()
    m.check()
    for whole, n in around:
        assert bool((whole[:offset] == 77).all()) and bool((whole[offset + n:] == 77).all())


@pytest.mark.gpu
def test_a_plan_for_other_moments_or_fewer_records():
    """What a plan does not hold is not gone through."""
    import ctypes
    import torch
    from ngraph_python_b200 import lib
    m = _Model([3000], 32, before=1)
    before = m.dev[0][0].clone()
    h = lib.AdamwHyper(*HYPER)
    lib.check(lib.raw().b2_adamw_step(m.plan.data_ptr(), m.chunks, 8, ctypes.byref(h), None, None, m.step_dev.data_ptr(), 0, 0))
    torch.cuda.synchronize()
    assert torch.equal(m.dev[0][0], before) and float(m.step_dev) == 1
    lib.check(lib.raw().b2_adamw_step(m.plan.data_ptr(), m.chunks + 1000, 32, ctypes.byref(h), None, None, m.step_dev.data_ptr(), m.seed, 0))
    m.expect()
    m.check()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_from_the_first_step_on(bits):
    """All zeros is the state before the first step; a gradient of zeros leaves it so."""
    m = _Model([300, 5000], bits, zero=True)
    for g in m.grads:
        g[0][:] = 0
        g[1].zero_()
    m.launch()
    m.expect()
    m.check()
    assert all(not s.any() for _, state in m.dev for s in state)
    for k in range(4):
        m.new_gradients(k)
        m.launch()
        m.expect()
        m.check()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("before", [999, 123456, 2 ** 24 - 2])
def test_late_steps_other_rates(bits, before):
    import torch
    m = _Model([1000, 77], bits, before=before)
    lr, scale = torch.tensor([0.01], device="cuda"), torch.tensor([0.125], device="cuda")
    hyper = (float(np.float32(0.01)), 0.8, 0.95, 1e-6, 0.0)
    m.launch((5.0,) + hyper[1:], lr, scale)
    m.expect(hyper, 0.125)
    m.check()


@pytest.mark.gpu
def test_no_tensors():
    """Only the number of the step moves."""
    m = _Model([], 32)
    m.launch()
    m.expect()
    m.check()
    m = _Model([0, 0], 8)
    m.launch()
    m.expect()
    m.check()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_and_replayed(bits):
    """Two models in one graph; the number of the step moves with every replay."""
    import torch
    models = [_Model([5000, 30], bits, seed=s) for s in (1, 2)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        for m in models:
            m.launch(stream=torch.cuda.current_stream().cuda_stream)
    for k in range(3):
        for m in models:
            m.new_gradients(10 + k)
        graph.replay()
        for m in models:
            m.expect()
            m.check()


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_where_they_are():
    """fp32 moments: a value's own.  8 bits: the moments of its 256 values."""
    for bits in (32, 8):
        m = _Model([1024], bits, before=3)
        g = m.grads[0]
        g[0][300] = np.inf
        g[1][300] = float("inf")
        m.launch()
        p = m.dev[0][0].cpu().numpy()
        assert np.array_equal(np.argwhere(~np.isfinite(p)), [[300]])
        m.launch()
        p = m.dev[0][0].cpu().numpy()
        bad = np.argwhere(~np.isfinite(p))[:, 0]
        assert 300 in bad and (len(bad) == 1 if bits == 32 else set(bad) == set(range(256, 512)))


@pytest.mark.gpu
def test_rounding_at_random_follows_a_falling_average():
    """Second moments that fall by 0.1 % a step under gradients of zero: rounded to nearest they would stay.  After 2000 steps
    v is 0.999^2000 = 0.135 of itself, its root 0.368.  A root's walk rounds to neighbours at most 1/8 apart: the sum of
    2000 roundings each of standard deviation at most sqrt(2^-3 * 0.0005) = 0.008 of the value is at most 0.36 of it for
    one value, 0.0056 for the mean of 4096; five of those and 0.01 for the first rounding."""
    import torch
    m = _Model([4096], 8, zero=True)
    codes, scales = m.dev[0][1][1], m.dev[0][1][3]
    codes.fill_(0x7e)                   # 448
    scales.fill_(1.0 / 448)
    for g in m.grads:
        g[1].zero_()
    # (a block's largest would move the scale alone: one value of each stays where it is)
    m.grads[0][1][::256] = 1.0
    codes.view(-1, 256)[:, 1:] = 0x76   # 224
    for _ in range(2000):
        m.launch()
    torch.cuda.synchronize()
    r = ao.E4M3[codes.cpu().numpy()].reshape(-1, 256) * scales.cpu().numpy()[:, None]
    assert abs(r[:, 1:].mean() / 0.5 - 0.999 ** 1000) <= 5 * 0.0056 + 0.01


def test_the_random_bits_are_spread_evenly():
    """2^20 hashes of neighbouring positions: each bit is set half the time within five standard deviations, and so is
    the parity of each pair of bits."""
    n = 1 << 20
    h = ao.mix(np.arange(n, dtype=np.uint32) ^ ao.mix(np.uint32(77)))
    room = 5 * 0.5 / np.sqrt(n)
    bits = [((h >> np.uint32(k)) & np.uint32(1)).astype(np.int8) for k in range(32)]
    for i in range(32):
        assert abs(bits[i].mean() - 0.5) < room
        for j in range(i):
            assert abs((bits[i] ^ bits[j]).mean() - 0.5) < room


def test_the_oracle_rounds_to_neighbours_with_the_right_chance():
    q = np.array([0.0, 2.0 ** -9, 448.0, 1.0, 1.0625, 300.0, 0.011, 0.001, -17.3], np.float32)
    for x in q:
        bits = np.arange(65536, dtype=np.uint32)
        got = ao.to_e4m3(np.full(65536, x, np.float32), bits)
        table = np.sort(ao.E4M3[:127])
        low = table[np.searchsorted(table, abs(x), side="right") - 1]
        high = table[min(np.searchsorted(table, abs(x), side="left"), 126)]
        assert set(np.unique(got)) <= {low, high}
        # (sixteen bits of the chance)
        assert abs(got.mean(dtype=np.float64) - abs(x)) <= (high - low) / 65536 + 1e-12


def test_second_moments_in_8_bits_settle_high():
    """Roots are rounded with their mean kept; squared they have the variance of each rounding on top.  A root that moves by d
    against a grid of distance D has a variance of f (1 - f) D^2 <= d D with f = d / D.  Under normal gradients d is
    E|g^2 / v - 1| / 2 = 0.48 of (1 - beta2) of the root on the average, and the grid, which goes with the block's largest, moves
    by at most as much downwards as that decays, 1/2, and upwards again as often: 1 together.  D is at most 1/8 of the root:
    v settles at most (0.48 + 1) / 8 = 18.5 % high.  At least, with d alone, D 1/16 and 1 - f above 1/2: 1.5 %.  (Seen: 4.9.)"""
    rng = np.random.RandomState(3)
    n, beta2 = 8192, 0.999
    zero = np.zeros(n, np.float32)
    state, v = (zero.astype(np.uint8), zero.astype(np.uint8), zero[:n // 256], zero[:n // 256]), np.zeros(n)
    for t in range(1, 501):
        g = rng.standard_normal(n).astype(np.float32)
        v = beta2 * v + (1 - beta2) * g.astype(np.float64) ** 2
        _, state = ao.step(zero, g, state, t, (1e-3, 0.9, beta2, 1e-8, 0.0), seed=5)
    held = (ao.E4M3[state[1]].reshape(-1, 256) * state[3][:, None]).astype(np.float64) ** 2
    assert 1.015 < held.mean() / v.mean() < 1.185


def _one(n=100, scales=True):
    from ngraph_python_b200 import lib
    t = (lib.AdamwTensor * 1)()
    t[0].param = t[0].grad = t[0].m = t[0].v = 256
    if scales:
        t[0].m_scales = t[0].v_scales = 256
    t[0].n = n
    return t


def test_refusals():
    from ngraph_python_b200 import lib
    raw = lib.raw()
    assert lib.adamw_plan_bytes(_one(2048 * 3 + 1), 8)[1] == 4
    for tensors, bits in ((_one(-1), 32), (_one(), 16), (_one(scales=False), 8)):
        with pytest.raises(lib.B200Error, match="error -1"):
            lib.adamw_plan_bytes(tensors, bits)
    for name in ("param", "grad", "m", "v"):
        t = _one()
        setattr(t[0], name, None)
        with pytest.raises(lib.B200Error, match="error -1"):
            lib.adamw_plan_bytes(t, 32)
    with pytest.raises(lib.B200Error, match="error -1"):
        lib.adamw_plan(_one(), 32, 256, 64)
    with pytest.raises(lib.B200Error, match="error -1"):
        lib.adamw_plan(_one(), 32, None, 1 << 20)
    good = dict(plan=256, chunks=1, bits=32, hyper=HYPER, step=256)
    for kw in (dict(plan=None), dict(chunks=-1), dict(bits=4), dict(step=None), dict(hyper=None), dict(hyper=(1e-3, 1.0, 0.9, 1e-8, 0)),
               dict(hyper=(1e-3, 0.9, -0.1, 1e-8, 0)), dict(hyper=(float("nan"), 0.9, 0.9, 1e-8, 0)), dict(hyper=(1e-3, 0.9, 0.9, -1.0, 0))):
        a = dict(good, **kw)
        h = None if a["hyper"] is None else ctypes.byref(lib.AdamwHyper(*a["hyper"]))
        with pytest.raises(lib.B200Error, match="error -1"):
            lib.check(raw.b2_adamw_step(a["plan"], a["chunks"], a["bits"], h, None, None, a["step"], 0, 0))


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_overlap_are_refused(bits):
    """Of two tensors of 600 values one address at a time moves into another range by a byte, or out of it."""
    from ngraph_python_b200 import lib
    names = ("param", "grad", "m", "v") + (("m_scales", "v_scales") if bits == 8 else ())
    size = dict.fromkeys(names, 2400)
    if bits == 8:
        size.update(m=600, v=600, m_scales=12, v_scales=12)
    at, place = 1 << 20, {}
    for k in range(2):
        for name in names:
            place[k, name] = at
            at += 8192
    def message(moved, to):
        t = (lib.AdamwTensor * 3)()
        for k in range(2):
            t[k].n = 600
            for name in names:
                setattr(t[k], name, to if (k, name) == moved else place[k, name])
        with pytest.raises(lib.B200Error) as e:      # (addresses of nothing: refused in any case)
            lib.adamw_plan(t, bits, 256, 1 << 20)
        return "overlap" in str(e.value)
    for moved in place:
        for other in place:
            if moved == other:
                continue
            both_read = moved[1] == other[1] == "grad"
            for to, overlap in ((place[other], True), (place[other] + size[other[1]] - 1, True), (place[other] + size[other[1]], False),
                                (place[other] - size[moved[1]] + 1, True), (place[other] - size[moved[1]], False)):
                assert message(moved, to) == (overlap and not both_read), (moved, other, to - place[other])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_plan_in_the_memory_of_a_tensor_is_refused(bits):
    """A step would write over the addresses that it goes by."""
    from ngraph_python_b200 import lib
    names = ("param", "grad", "m", "v") + (("m_scales", "v_scales") if bits == 8 else ())
    t = (lib.AdamwTensor * 1)()
    t[0].n = 40000
    size = dict.fromkeys(names, 160000)
    if bits == 8:
        size.update(m=40000, v=40000, m_scales=628, v_scales=628)
    for k, name in enumerate(names):
        setattr(t[0], name, (k + 1) << 20)
    need, _ = lib.adamw_plan_bytes(t, bits)
    for name in names:
        at = getattr(t[0], name)
        for plan, overlap in ((at, True), (at + size[name] - 4, True), (at + size[name], False), (at - need + 4, True), (at - need, False)):
            with pytest.raises(lib.B200Error) as e:      # (addresses of nothing: refused in any case)
                lib.adamw_plan(t, bits, plan, need)
            assert ("overlap" in str(e.value)) == overlap


@pytest.mark.parametrize("bits", [32, 8])
def test_addresses_between_two_values_are_refused(bits):
    from ngraph_python_b200 import lib
    names = ("param", "grad", "m", "v") + (("m_scales", "v_scales") if bits == 8 else ())

    def message(moved, by):
        t = (lib.AdamwTensor * 2)()
        for k in range(2):
            t[k].n = 100
            for j, name in enumerate(names):
                setattr(t[k], name, (1 << 20) + 4096 * (8 * k + j) + (by if (k, name) == moved else 0))
        with pytest.raises(lib.B200Error) as e:      # (addresses of nothing: refused in any case)
            lib.adamw_plan(t, bits, 256, 1 << 20)
        return str(e.value)
    for moved in [(k, name) for k in range(2) for name in names]:
        for by in (0, 1, 2, 3, 4, 8):
            # (moments in 8 bits are bytes)
            assert ("tensor %d lies between" % moved[0] in message(moved, by)) == (by % 4 != 0 and not (bits == 8 and moved[1] in "mv"))
    h = lib.AdamwHyper(*HYPER)
    for k in range(3):
        at = [256, 512, 768]
        at[k] += 2
        with pytest.raises(lib.B200Error, match="between two addresses"):
            lib.check(lib.raw().b2_adamw_step(4096, 1, bits, ctypes.byref(h), at[0], at[1], at[2], 0, 0))


@pytest.mark.gpu
def test_a_plan_is_not_made_in_a_recording():
    import torch
    from ngraph_python_b200 import lib
    m = _Model([64], 32)
    x = torch.zeros((4,), device="cuda")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        x.add_(1)
        with pytest.raises(lib.B200Error, match="captured"):
            lib.adamw_plan(m.tensors, 32, m.plan.data_ptr(), m.plan.numel(), torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert float(x[0]) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_numbers_and_plans_in_host_memory_are_refused(bits):
    import torch
    from ngraph_python_b200 import lib
    m = _Model([300, 5], bits)
    host = np.full((4096,), 7.0, np.float32)
    good = dict(plan=m.plan.data_ptr(), lr=None, scale=None, step=m.step_dev.data_ptr())

    def step(**kw):
        a = dict(good, **kw)
        h = lib.AdamwHyper(*HYPER)
        lib.check(lib.raw().b2_adamw_step(a["plan"], m.chunks, bits, ctypes.byref(h), a["lr"], a["scale"], a["step"], m.seed,
                                          torch.cuda.current_stream().cuda_stream))
    for name in good:
        with pytest.raises(lib.B200Error, match="memory"):
            step(**{name: host.ctypes.data})
    # numbers in page-locked memory are read
    numbers = torch.tensor([HYPER[0], 1.0]).pin_memory()
    step(lr=numbers.data_ptr(), scale=numbers.data_ptr() + 4)
    m.expect((float(np.float32(HYPER[0])),) + HYPER[1:])
    m.check()
    assert (host == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
def test_gradients_in_page_locked_memory_are_read(bits, offset):
    import torch
    from ngraph_python_b200 import lib
    m = _Model([5000, 7, 2048], bits, offset=offset, before=2)
    held = []
    for x, g in zip(m.tensors, m.grads):
        t = torch.zeros((g[0].size + offset,)).pin_memory()
        t[offset:] = torch.from_numpy(g[0])
        held.append(t)
        x.grad = t.data_ptr() + 4 * offset
    lib.adamw_plan(m.tensors, bits, m.plan.data_ptr(), m.plan.numel(), torch.cuda.current_stream().cuda_stream)
    m.launch()
    m.expect()
    m.check()
    pageable, locked = np.zeros(5000, np.float32), torch.zeros((5000,)).pin_memory()
    for name, data in (("grad", pageable.ctypes.data), ("param", locked.data_ptr())):
        kept = getattr(m.tensors[0], name)
        setattr(m.tensors[0], name, data)
        with pytest.raises(lib.B200Error, match="memory"):
            lib.adamw_plan(m.tensors, bits, m.plan.data_ptr(), m.plan.numel(), torch.cuda.current_stream().cuda_stream)
        setattr(m.tensors[0], name, kept)
