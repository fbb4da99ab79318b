"""Steps of orthogonalised updates in a graph: of gradients that replicas exchange, and of a projection's weight as one matrix."""
import numpy as np
import pytest

import ngraph_python_b200 as ng
from oracle import muon_oracle as mo

HALF = 2.0 ** -24


def _transformer(**kw):
    return ng.transformers.make_transformer_factory("b200", **kw)()


def _axes(**lengths):
    return [ng.make_axis(n, name=k) for k, n in lengths.items()]


def test_muon_and_adamw_of_gradients_that_replicas_exchange():
    """Both steps come behind the exchanges of all their gradients, results of norms of heads among them, and read what these leave."""
    class Two(object):
        size, rank = 2, 0
    T, F, H, D = _axes(T=16, F=12, H=3, D=8)
    x, d = ng.placeholder([T, F]), ng.placeholder([T, H, D])
    w, scale = ng.variable([F, H, D], initial_value=1), ng.variable([D], initial_value=1)
    q = ng.dot(x, w)
    out = ng.head_norm([q], [scale], heads=[H], features=D, rotation=ng.Rotation(T))
    g = ng.head_norm_grad([d], out)
    shared = [ng.allreduce(ng.dot(x, g["x"][0]), "mean"), ng.allreduce(g["weight"][0])]
    t = _transformer(plan_only=True, comm=Two())
    comp = t.computation([ng.muon([w], shared[:1], lr=0.1), ng.adamw([scale], shared[1:], lr=0.1)], x, d)
    t.initialize()
    kinds = [s.kind for s in comp.steps]
    assert sorted(kinds) == sorted(["gemm", "head_norm", "head_norm_grad", "gemm", "comm", "comm", "muon", "adamw"])
    exchanges = [s for s in comp.steps if s.kind == "comm"]
    for kind in ("muon", "adamw"):
        step = comp.steps[kinds.index(kind)]
        mine = [s for s in exchanges if s.arena_buffer in [v.buffer for v in step.gradients]]
        assert len(mine) == len(step.gradients) == 1 and comp.steps.index(mine[0]) < comp.steps.index(step)
        assert mine[0].arena_buffer in [v.buffer for v in step.in_views]        # (what a step reads is waited for)
        made = [k for k, s in enumerate(comp.steps) if s.kind != "comm" and mine[0].arena_buffer in [v.buffer for v in s.out_views]]
        assert len(made) == 1 and made[0] < comp.steps.index(mine[0])
    assert sorted(s.reduce_func for s in exchanges) == ["mean", "sum"]


def _projection():
    """A product that makes heads, whose weight is one matrix of two axes, and the step over it."""
    T, F, H, D = _axes(T=40, F=96, H=5, D=24)
    C = ng.make_axis(5 * 24, name="C")
    rng = np.random.RandomState(4)
    value = rng.standard_normal((96, 120)).astype(np.float32)
    w, x, d = ng.variable([F, C], initial_value=value), ng.placeholder([T, F]), ng.placeholder([T, H, D])
    heads = ng.dot(x, ng.reshape(w, [F, H, D]))                         # [T, H, D]
    gradient = ng.reshape(ng.dot(x, d), [F, C])
    return w, value, [x, d], heads, gradient, ng.muon([w], [gradient], lr=0.5)


def test_a_projections_weight_as_one_matrix_takes_no_copies():
    w, _, args, heads, gradient, step = _projection()
    t = _transformer(plan_only=True)
    comp = t.computation([heads, step], *args)
    t.initialize()
    assert sorted(s.kind for s in comp.steps) == ["gemm", "gemm", "muon"]
    assert step.shapes == [(1, 96, 120)]


@pytest.mark.gpu
def test_a_projections_weight_as_one_matrix():
    """The update of the 96 x 120 matrix, from the step's own gradient: off by what its roundings add up to (the oracle's), and
    the rounding of the weights' two products and their difference."""
    w, value, args, heads, gradient, step = _projection()
    t = _transformer()
    comp = t.computation([heads, gradient, step], *args)
    rng = np.random.RandomState(5)
    mean = np.zeros((96, 120))
    for k in range(3):
        x, d = rng.standard_normal((40, 96)).astype(np.float32), rng.standard_normal((40, 5, 24)).astype(np.float32)
        y, g, count = comp(x, d)
        terms = np.einsum("tf,fhd->thd", np.abs(x).astype(np.float64), np.abs(value).reshape(96, 5, 24))
        assert np.all(np.abs(y - np.einsum("tf,fhd->thd", x.astype(np.float64), value.reshape(96, 5, 24))) <= 100 * HALF * terms)    # (96 terms)
        assert float(np.ravel(count)[0]) == k + 1
        u, mean = mo.update(np.asarray(g, np.float64).reshape(96, 120), mean)
        want = value - 0.5 * mo.orthogonal(u)[0]
        held = np.array(t.device_tensor(w).get(None))
        off = np.sqrt(np.sum((held - want) ** 2))
        assert off <= 0.5 * mo.spread(u) + 3 * HALF * np.sqrt(np.sum(value.astype(np.float64) ** 2) + np.sum(want ** 2)), off
        value, mean = held, np.array(t.device_tensor(step.states[0]).get(None)).astype(np.float64)
        if k == 0:
            comp.capture()
    t.close()
