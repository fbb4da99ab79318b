"""Orthogonalised updates of gradients whose norm, or its reciprocal, is no fp32 number, and where the numbers of a step may lie."""
import ctypes

import numpy as np
import pytest

from ngraph_python_b200 import lib
from oracle import muon_oracle as mo
from tests.test_muon_operator import HALF, STEP, _Step


@pytest.mark.gpu
@pytest.mark.parametrize("r,c", [(70, 90), (90, 70), (300, 400), (64, 769)])
def test_norms_beyond_fp32(r, c):
    """The same directions whatever their size: whole numbers of 12 bits times a power of two, without a mean before them, so that
    u is exact and the update that of size one but for the rounding of the factors.  As far off as products in fp32 are at most
    (see the tests of the orthogonalised matrix itself)."""
    rng = np.random.RandomState(r + c)
    whole = rng.randint(-2047, 2048, (r, c)).astype(np.float32)
    sizes = [2.0 ** e for e in (0, 115, 116, -126, -138, -149)]       # largest 2^127; the last two are below the normal numbers
    data = [dict(param=np.zeros((r, c), np.float32), grad=np.ldexp(whole, int(np.log2(s))).astype(np.float32), mean=np.zeros((r, c), np.float32)) for s in sizes]
    for d, s in zip(data, sizes):
        assert np.array_equal(d["grad"].astype(np.float64), whole.astype(np.float64) * s)
    step = _Step(data, hyper=dict(lr=1.0, weight_decay=0.0, momentum=0.0, nesterov=0, eps=0.0))
    step()
    got = [g["param"].astype(np.float64) for g in step.get()]
    x = whole.astype(np.float64)
    x /= np.sqrt(np.sum(x * x))
    want, _ = mo.orthogonal(x)
    # (fp32's own iteration, four times as far at most, and the roundings of the factor and of the move)
    y = (x.T if r > c else x).astype(np.float32)
    for _ in range(5):
        a = y @ y.T
        y = np.float32(mo.A) * y + (np.float32(mo.B) * a + np.float32(mo.C) * (a @ a)) @ y
    plain = np.sqrt(np.sum(((y.T if r > c else y) - want) ** 2))
    limit = 4 * plain + 8 * HALF * np.sqrt(np.sum(want ** 2))
    for s, g in zip(sizes, got):
        assert np.sqrt(np.sum((g + want) ** 2)) <= limit, (s, np.sqrt(np.sum((g + want) ** 2)), limit)


def test_numbers_in_the_memory_of_a_step_are_refused():
    """The rate, the scale, the count and the status: none in the plan or the scratch, which the step writes, and what is written not
    in the place of another."""
    m = (lib.MuonMatrix * 1)()
    m[0].param, m[0].grad, m[0].mean, m[0].rows, m[0].cols, m[0].decay, m[0].scale = 1 << 20, 2 << 20, 3 << 20, 200, 300, 1.0, 1.0
    sizes, h = lib.muon_plan_sizes(m), lib.MuonHyper(**STEP)
    plan, scratch, apart = 1 << 33, 1 << 34, [(1 << 35) + 256 * i for i in range(4)]

    def said(*numbers):
        rc = lib.raw().b2_muon_step(plan, ctypes.byref(sizes), ctypes.byref(h), *numbers[:3], scratch, sizes.scratch_bytes, numbers[3], None)
        return lib.raw().b2_last_error().decode() if rc == -1 else ""
    assert "lies in" not in said(*apart)
    for i in range(4):
        for place in (plan, plan + sizes.plan_bytes - 4, scratch, scratch + sizes.scratch_bytes - 4):
            assert "in the plan or the scratch" in said(*(apart[:i] + [place] + apart[i + 1:])), i
        for place in (plan - 4, plan + (sizes.plan_bytes + 3) // 4 * 4, scratch - 4, scratch + (sizes.scratch_bytes + 3) // 4 * 4):
            assert "lies in" not in said(*(apart[:i] + [place] + apart[i + 1:])), i
    for i, j in ((0, 2), (1, 2), (2, 3), (0, 3), (1, 3)):
        numbers = list(apart)
        numbers[j] = numbers[i]
        assert "in the place of" in said(*numbers), (i, j)
    assert "lies in" not in said(apart[0], apart[0], apart[2], apart[3])        # (one number for both that are only read)
