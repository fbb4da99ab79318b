"""How exact the orthogonalised update is: the update alone, onto a param of zeros at a rate of one, of matrices of all shapes and of
plans whose tiles are wide, or of several groups of matrices.

The oracle says how far the result is where every rounding is as large as it can be, with signs by chance; that is granted, and
the two roundings of the move.  What one part of an operand instead of two, or two of the three products, would make of it is
far outside (see the tests of the bound)."""
import numpy as np
import pytest

from ngraph_python_b200 import lib
from oracle import muon_oracle as mo
from tests.test_muon_operator import HALF, SHAPES, _data, _Step

ALONE = dict(lr=1.0, weight_decay=0.0)


def _alone(r, c, seed=0, kind="gauss"):
    d = _data(r, c, seed, "few" if kind == "few" else "gauss")
    d["param"][:] = 0
    if kind == "rows":                  # rows over six decades
        by = np.float32(10.0) ** np.linspace(-3, 3, r).astype(np.float32)[:, None]
        d["grad"], d["mean"] = d["grad"] * by, d["mean"] * by
    return d


def _want(d):
    """(the update, how far it may be off)"""
    x, _ = mo.update(d["grad"], d["mean"])
    want, _ = mo.orthogonal(x)
    return want, mo.spread(x) + 2 * HALF * np.sqrt(np.sum(want ** 2))


def _off(param, want):
    return np.sqrt(np.sum((param.astype(np.float64) + want) ** 2))


def _plan_of(shapes):
    m = (lib.MuonMatrix * sum(n for n, _, _ in shapes))()
    k = 0
    for n, r, c in shapes:
        for _ in range(n):
            x = m[k]
            x.param = x.grad = x.mean = 256
            x.rows, x.cols, x.decay, x.scale = r, c, 1.0, 1.0
            k += 1
    return lib.muon_plan_tiles(m)


# (count, rows, columns); groups; the widths, in blocks of columns, that tiles of A, of B and of x have
PLANS = [([(30, 700, 1000), (30, 1000, 700)], 1, ({1, 3, 4}, {1, 3, 4}, {3, 4})),
         ([(8, 640, 1920), (8, 1920, 640)], 1, ({2, 4}, {2, 4}, {2, 4})),
         ([(40, 130, 4100)], 1, ({1}, {1, 2}, {1, 4})),
         ([(250, 321, 450), (250, 450, 321)], 4, ({2, 4}, {2, 4}, {2, 4})),
         ([(50, 1000, 1000), (300, 256, 300), (20, 77, 77), (5, 1300, 500)], 3, ({2, 4}, {2, 4}, {1, 4}))]


@pytest.mark.parametrize("shapes,groups,widths", PLANS, ids=str)
def test_the_plans_have_wide_tiles_and_groups(shapes, groups, widths):
    found, tiles = _plan_of(shapes)
    assert found == groups
    assert tuple(set(w + 1 for w, n in enumerate(t) if n) for t in tiles) == widths


def test_tiles_of_small_matrices_and_refusals():
    assert _plan_of([]) == (0, [[0] * 4] * 3)
    assert _plan_of([(3, 64, 64)])[1] == [[0] * 4] * 3
    with pytest.raises(lib.B200Error, match="sides"):
        _plan_of([(1, -1, 4)])
    assert lib.raw().b2_muon_plan_tiles(None, 0, None) == -1


BOUND = [(r, c) for r, c in SHAPES if min(r, c) >= 64]


@pytest.mark.parametrize("r,c", BOUND)
@pytest.mark.parametrize("kind", ["gauss", "few", "rows"])
def test_the_bound_tells_parts_and_products_that_are_missing(r, c, kind):
    d = _alone(r, c, kind=kind)
    want, limit = _want(d)
    x, _ = mo.update(d["grad"], d["mean"])
    off = lambda **kw: np.sqrt(np.sum((mo.emulated(x, **kw) - want) ** 2))  # noqa: E731
    assert off() <= limit
    assert off(products=2) > 5 * limit and off(parts=1) > 5 * limit


@pytest.mark.gpu
@pytest.mark.parametrize("r,c", SHAPES + [(640, 1920), (1920, 640), (700, 1000), (513, 2049)])
@pytest.mark.parametrize("kind", ["gauss", "few", "rows"])
def test_the_update_of_one_matrix(r, c, kind):
    d = _alone(r, c, kind=kind)
    s = _Step([d], hyper=ALONE)
    s()
    want, limit = _want(d)
    off = _off(s.get()[0]["param"], want)
    assert off <= limit, (off, limit)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes,groups,widths", PLANS, ids=str)
def test_the_updates_of_a_plan(shapes, groups, widths):
    """Two matrices of each shape and of unlike kinds, again and again; two steps, of which the second finds the scratch used."""
    data = []
    for n, r, c in shapes:
        two = [_alone(r, c, k, kind) for k, kind in enumerate(("gauss", "rows"))]
        data.append([two[i % 2] for i in range(n)])
    wants = [[_want(d) for d in of[:2]] for of in data]
    flat = [d for of in data for d in of]
    s = _Step(flat, hyper=ALONE)
    for again in range(2):
        if again:
            for on, d in zip(s.all, flat):
                on["param"][:d["param"].size].zero_()
                on["mean"][:d["mean"].size].copy_(s.torch.from_numpy(d["mean"].ravel()))
        s()
        got, k = s.get(), 0
        for of, want in zip(data, wants):
            for i in range(len(of)):
                off = _off(got[k]["param"], want[i % 2][0])
                assert off <= want[i % 2][1], (of[0]["param"].shape, i, off, want[i % 2][1])
                k += 1
