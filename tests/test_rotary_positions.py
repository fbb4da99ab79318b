"""Positions of rotations whose values go beyond those of earlier calls, in a flex16 transformer, and frequencies to the last bit."""
import numpy as np
import pytest

from ngraph_python_b200 import lib
from ngraph_python_b200 import op_graph as ng
from ngraph_python_b200.transformers import make_transformer_factory
from oracle import heads_oracle as ho


def _transformer(**kw):
    return make_transformer_factory("b200", **kw)()


def _axes(**lengths):
    return [ng.make_axis(n, name=k) for k, n in lengths.items()]


def test_which_positions_a_flex_transformer_holds_in_fp32():
    """Placeholders that rotations alone read, through views too, in whichever of its computations; others are flex16 tensors."""
    T, B, H, D = _axes(T=6, B=2, H=2, D=8)
    for case in ("alone", "sliced", "added", "added elsewhere", "rotated itself", "variable"):
        x = ng.placeholder([B, T, H, D])
        p = ng.variable([T], initial_value=1) if case == "variable" else ng.placeholder([T, D]) if case in ("sliced", "rotated itself") else ng.placeholder([T])
        at = ng.tensor_slice(p, [slice(None), 3]) if case in ("sliced", "rotated itself") else p
        r = ng.Rotation(at)
        y = ng.rotary(x, r, heads=H, features=D)
        wanted, more = [y, ng.rotary_grad(y, y)], []
        if case == "added":
            wanted.append(p + p)
        if case == "added elsewhere":
            more = [p + p]
        if case == "rotated itself":
            wanted.append(ng.rotary(p, ng.Rotation(T), heads=None, features=D))
        t = _transformer(flex=True, plan_only=True)
        comp = t.computation(wanted, x, p) if case != "variable" else t.computation(wanted, x)
        if more:
            t.computation(more, p)
        t.initialize()
        assert t._buffer_of(p).flex == (case not in ("alone", "sliced")), case
        assert t._buffer_of(x).flex and t._buffer_of(y).flex
        assert all(s.in_views[1].buffer.flex == t._buffer_of(p).flex for s in comp.steps if s.kind == "rotary" and len(s.in_views) > 1)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("order", ["T", "BT", "TB"])
def test_positions_that_outgrow_the_first_calls_in_flex16(pairs, order):
    """Positions near zero first, then beyond 16 bits, from the host and from the device, in calls one by one and recorded.

    The largest of the values, one, lies alone in its pair, so that no result is larger than the first call's, at position zero.  A
    value is cut to a step of 2^-14 -- a rotated one moves by both of its pair's -- and a result is off by half a step of its own, where
    the exponent leaves room for up to three deviations of the largest ones: a step of at most 2^-12."""
    import torch
    T, B, H, D = ng.make_axis(9, name="T"), ng.make_axis(2, name="B"), ng.make_axis(3, name="H"), ng.make_axis(16, name="D")
    ax = dict(T=T, B=B)
    rng = np.random.RandomState(3)
    v = rng.uniform(-0.6, 0.6, (2, 9, 3, 16)).astype(np.float32)
    v[0, 4, 1, :] = 0
    v[0, 4, 1, 0] = 1
    shape = [ax[c].length for c in order]
    x, at = ng.placeholder([B, T, H, D]), ng.placeholder([ax[c] for c in order])
    t = _transformer(flex=True)
    comp = t.computation(ng.rotary(x, ng.Rotation(at, pairs=pairs, base=100000.0), heads=H, features=D), x, at)
    for call, most in enumerate((1, 5, 900, 40000, 1 << 20, 1 << 24, 3, 1 << 22)):
        p = rng.randint(0, most, shape).astype(np.float32)
        p.flat[-1] = max(most - 1, 0)
        given = torch.from_numpy(p).cuda() if call % 2 else p
        out = comp(v, given)
        rows = p.T if order == "TB" else np.broadcast_to(p, (2, 9))
        angle = rows.reshape(18)[:, None].astype(np.float64) * ho.frequencies(16, base=100000.0)
        want, _ = ho.rotate(v.reshape(18, 3, 16), angle, 16, pairs == "neighbours")
        assert np.abs(out.reshape(18, 3, 16) - want).max() <= 2 * 2.0 ** -14 + 2.0 ** -13, (call, most)
        if call == 2:
            comp.capture()
    t.close()


PI = "3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803"


def _exact_turns(d, base=10000.0, scaling="none", factor=1.0, original=1.0, low=1.0, high=32.0):
    """Turns a position of each pair, in 80 digits."""
    import decimal
    with decimal.localcontext(decimal.Context(prec=80)):
        D = decimal.Decimal
        base, factor, original, low, high, found = D(base), D(factor), D(original), D(low), D(high), []
        if scaling == "base" and d > 2:
            base = base * factor ** (D(d) / D(d - 2))
        for i in range(d // 2):
            f = base ** (D(-2 * i) / D(d)) / (2 * D(PI))
            if scaling == "linear":
                f /= factor
            if scaling == "parts":
                keep = min(max((original * f - low) / (high - low), D(0)), D(1))
                f = keep * f + (1 - keep) * f / factor
            found.append(f)
        return [int((f % 1 * 2 ** 64).to_integral_value()) for f in found], [float(f) for f in found]


@pytest.mark.parametrize("d", [2, 6, 40, 128, 256, 1024])
@pytest.mark.parametrize("scaling", ["none", "linear", "base", "parts"])
@pytest.mark.parametrize("base", [500.0, 10000.0, 1e6, 0.25])
def test_frequencies_to_64_bits(d, scaling, base):
    """A fraction of a turn is rounded to 2^-64 of one (half a step), and the operations before it round to 64 bits each: a power by a
    step (2^-63 of itself), its exponent by half a step times the logarithm of the base, the others by half a step.  With
    up to eight of them, and a power and a logarithm of 14 within one, that is 2^-59 of a frequency."""
    kw = dict(base=base, scaling=scaling, factor=8.0, original=300.0, low=1.0, high=20.0)
    want, size = _exact_turns(d, **kw)
    got = [int(v) for v in lib.rotary_turns(d, **kw).numpy().view(np.uint64)]
    for g, w, f in zip(got, want, size):
        off = (g - w + (1 << 63)) % (1 << 64) - (1 << 63)
        assert abs(off) <= 1 + f * 2.0 ** 5, (off, f)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 21, 520])
def test_the_largest_fp32_positions_that_64_bits_hold(D):
    """Whole numbers up to the last fp32 value below 2^63, and -2^63 itself; beyond, a rotation is NaN.  (Off as any rotation is.)"""
    import ctypes
    import torch
    p = np.array([np.nextafter(np.float32(2.0 ** 63), np.float32(0)), 9.21e18, -2.0 ** 63, 2.0 ** 63, np.nextafter(np.float32(-2.0 ** 63), np.float32(-np.inf))], np.float32)
    x = np.random.RandomState(0).standard_normal((5, 2, D)).astype(np.float32)
    rotary = D // 2 * 2
    turns = lib.rotary_turns(rotary)
    at, on, turns_on = torch.from_numpy(p).cuda(), torch.from_numpy(x).cuda(), turns.cuda()
    out = torch.empty_like(on)
    a = lib.HeadsArgs(rows=5, head_dim=D, rotary_dim=rotary, parts=1, turns=turns_on.data_ptr(), positions=at.data_ptr(), position_kind=lib.IDX_F32,
                      position_count=5, position_group=1, amplitude=1.0)
    a.part[0] = lib.HeadsPart(x=on.data_ptr(), out=out.data_ptr(), x_row=2 * D, x_head=D, out_row=2 * D, out_head=D, heads=2)
    lib.check(lib.raw().b2_rotary(ctypes.byref(a), 0, None, None, None, 0, None))
    got = out.cpu().numpy()
    want, size = ho.rotate(x[:3], ho.angles(np.array([int(v) for v in p[:3]]), turns.numpy()), rotary, False)
    assert np.all(np.abs(got[:3] - want) <= 6 * 2.0 ** -24 * size)
    assert np.isnan(got[3:, :, :rotary]).all() and np.array_equal(got[..., rotary:], x[..., rotary:])
