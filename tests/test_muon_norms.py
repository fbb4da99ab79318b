"""Orthogonalised updates of gradients whose norm, or its reciprocal, is no fp32 number."""
import numpy as np
import pytest

from oracle import muon_oracle as mo
from tests.test_muon_operator import HALF, _Step


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
