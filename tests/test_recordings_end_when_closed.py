"""A transformer's recorded computations hold their graphs until it is closed, not until the garbage collector comes by: a graph that
is destroyed while another is recorded ends that recording with an error."""
import gc
import weakref

import numpy as np
import pytest

import ngraph_python_b200 as ng


@pytest.mark.gpu
def test_recordings_end_when_closed():
    A = ng.make_axis(8, name="A")
    x = ng.placeholder([A])
    t = ng.transformers.make_transformer_factory("b200")()
    comp = t.computation(x * 2.0, x)
    v = np.arange(8, dtype=np.float32)
    comp(v)
    comp.capture()
    assert np.array_equal(comp(v), 2 * v)
    held = [weakref.ref(g) for g in comp._graphs if g is not None]
    collecting = gc.isenabled()
    gc.disable()
    try:
        assert held and all(g() is not None for g in held)
        t.close()
        assert all(g() is None for g in held)
    finally:
        if collecting:
            gc.enable()
    from ngraph_python_b200 import lib
    with pytest.raises(lib.B200Error, match="closed"):
        comp(v)
