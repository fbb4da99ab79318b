"""Positions of rotations whose values go beyond those of earlier calls, in a flex16 transformer, and beyond what other types name."""
import numpy as np
import pytest

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
