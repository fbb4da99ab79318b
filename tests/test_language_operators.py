"""The language-model operators as ops of a graph: lookups with a scale, norms between blocks, AdamW, each against
numpy and together in a training step, step by step and recorded."""
import numpy as np
import pytest

import ngraph_python_b200 as ng
from oracle import adamw_oracle as ao
from oracle import flex_oracle as fx
from oracle import norm_oracle as no

ngt = ng.transformers


def _transformer(**kw):
    return ngt.make_transformer_factory("b200", **kw)()


def _axes(**lengths):
    return [ng.make_axis(n, name=k) for k, n in lengths.items()]


# ---- construction ------------------------------------------------------------------------------------
def test_axes_and_refusals_of_the_ops():
    V, F, T, B = _axes(V=11, F=6, T=5, B=3)
    table, idx = ng.variable([V, F], initial_value=0), ng.placeholder([B, T])
    e = ng.embedding(table, idx, scale=2.0)
    assert e.axes == ng.make_axes([B, T, F])
    g = ng.embedding_grad(ng.placeholder([B, T, F]), e)
    assert g.axes == table.axes
    x, u, w = ng.placeholder([B, T, F]), ng.placeholder([B, T, F]), ng.variable([F], initial_value=1)
    stream, out = ng.residual_norm(x, u, w, axes=[F], gate=ng.placeholder([B, T]))
    assert stream.axes == out.axes == ng.make_axes([B, T, F])
    assert ng.residual_norm(x, u, None, axes=[F])[1] is None
    grads = ng.residual_norm_grad(out, d_out=ng.placeholder([B, T, F]))
    assert {k: v.axes for k, v in grads.items()} == dict(residual=x.axes, block=x.axes, gate=ng.make_axes([B, T]), weight=w.axes)
    step = ng.adamw([w, table], [grads["weight"], g], lr=0.1, state_bits=8, no_decay=[w])
    assert [len(s) for s in step.states] == [4, 4] and step.decayed == [False, True]
    three = ng.variable([V, F, T], initial_value=0)
    for build in (lambda: ng.embedding(three, idx), lambda: ng.embedding(table, ng.placeholder([F])), lambda: ng.embedding(table, ng.placeholder([])),
                  lambda: ng.embedding_grad(ng.placeholder([B, F]), e), lambda: ng.embedding_grad(x, out),
                  lambda: ng.rms_norm(x, w, axes=[V]), lambda: ng.rms_norm(x, ng.placeholder([T]), axes=[F]), lambda: ng.rms_norm(x, None, axes=[F]),
                  lambda: ng.residual_norm(x, ng.placeholder([T, F]), w, axes=[F]), lambda: ng.residual_norm(x, u, w, axes=[F], gate=ng.placeholder([B])),
                  lambda: ng.residual_norm(x, u, w, axes=[]), lambda: ng.residual_norm(x, None, w, axes=[F], gate=w),
                  lambda: ng.residual_norm(x, None, w, axes=[F], residual_scale=0.5), lambda: ng.rms_norm(x, w, axes=[F], eps=-1.0),
                  lambda: ng.residual_norm_grad(out), lambda: ng.residual_norm_grad(out, d_stream=x), lambda: ng.residual_norm_grad(x, d_out=x),
                  lambda: ng.residual_norm_grad(out, d_out=ng.placeholder([T, F])),
                  lambda: ng.adamw([w], [], lr=0.1), lambda: ng.adamw([w], [x], lr=0.1), lambda: ng.adamw([w, w], [w, w], lr=0.1),
                  lambda: ng.adamw([out], [x], lr=0.1), lambda: ng.adamw([w], [w], lr=0.1, state_bits=16),
                  lambda: ng.adamw([w], [w], lr=0.1, no_decay=[table]), lambda: ng.adamw([w], [w], lr=x), lambda: ng.adamw([w], [w], lr=0.1, beta1=1.0)):
        with pytest.raises(ValueError):
            build()


def test_flex_transformers_refuse_norms_and_adamw():
    F, T = _axes(F=8, T=4)
    x, w = ng.placeholder([T, F]), ng.variable([F], initial_value=1)
    for op in (ng.rms_norm(x, w, axes=[F]), ng.adamw([w], [ng.placeholder([F])], lr=0.1)):
        t = _transformer(flex=True, plan_only=True)
        t.computation(op, x)
        with pytest.raises(ValueError, match="not flex16"):
            t.initialize()


@pytest.mark.parametrize("flex,rows", [(True, 32769), (False, (1 << 24) + 1)])
def test_an_index_that_cannot_name_every_row_is_refused(flex, rows):
    V, F, T = _axes(V=rows, F=1, T=2)
    idx = ng.placeholder([T])
    t = _transformer(flex=flex, plan_only=True)
    t.computation(ng.embedding(ng.placeholder([V, F]), idx), idx)
    with pytest.raises(ValueError, match="at most"):
        t.initialize()


def test_steps_of_a_plan():
    """One step each, and no copy of operands that lie as they should -- rows of a wider tensor among them."""
    V, F, T = _axes(V=50, F=8, T=16)
    wide = ng.make_axis(24, name="F")
    table, idx, w = ng.variable([V, F], initial_value=0), ng.placeholder([T]), ng.variable([F], initial_value=1)
    e = ng.embedding(table, idx)
    u = ng.cast_axes(ng.tensor_slice(ng.placeholder([T, wide]), [slice(None), slice(8, 16)]), [T, F])
    stream, out = ng.residual_norm(e, u, w, axes=[F])
    grads = ng.residual_norm_grad(out, d_out=out)
    g = ng.embedding_grad(grads["residual"], e)
    t = _transformer(plan_only=True)
    comp = t.computation([ng.adamw([table, w], [g, grads["weight"]], lr=0.1), stream], idx)
    t.initialize()
    assert [s.kind for s in comp.steps] == ["embed", "norm", "norm_grad", "embed_grad", "adamw"]
    t = _transformer(plan_only=True)
    turned = ng.placeholder([F, T])
    comp = t.computation(ng.rms_norm(ng.axes_with_order(turned, [T, F]), w, axes=[F]), turned)
    t.initialize()
    assert [s.kind for s in comp.steps] == ["dimshuffle", "norm"]


def test_gradients_that_are_variables_of_the_step_are_copied_first():
    """The loss sum(x * y) has the gradients y and x."""
    A, B = _axes(A=5, B=4)
    x, y = ng.variable([A, B], initial_value=1), ng.variable([A, B], initial_value=2)
    r, g = ng.variable([], initial_value=0.1), ng.placeholder([A, B])
    for op, copies in ((ng.adamw([x, y], [y, x], lr=0.1), 2), (ng.adamw([x, y], [g, x], lr=0.1), 1), (ng.adamw([x], [y], lr=0.1), 0),
                       (ng.adamw([x], [x], lr=0.1), 1), (ng.adamw([r, x], [ng.tensor_slice(x, [0, 0]), g], lr=r, grad_scale=r), 2)):
        t = _transformer(plan_only=True)
        comp = t.computation(op, g)
        t.initialize()
        assert [s.kind for s in comp.steps] == ["dimshuffle"] * copies + ["adamw"]
        step = comp.steps[-1]
        written = set(t._buffer_of(v) for v in op.written())
        assert [v.buffer for v in step.out_views] == [t._buffer_of(v) for v in op.written()]
        assert not any(v is not None and v.buffer in written for v in step.gradients + step.numbers)


def test_adamw_of_gradients_that_replicas_exchange():
    """The step comes behind the exchanges of all its gradients, results of norms among them, and reads what they leave."""
    class Two(object):
        size, rank = 2, 0
    V, F, T = _axes(V=50, F=8, T=16)
    table, idx, w, d = ng.variable([V, F], initial_value=0), ng.placeholder([T]), ng.variable([F], initial_value=1), ng.placeholder([T, F])
    e = ng.embedding(table, idx)
    grads = ng.residual_norm_grad(ng.rms_norm(e, w, axes=[F]), d_out=d)
    shared = [ng.allreduce(ng.embedding_grad(grads["residual"], e)), ng.allreduce(grads["weight"], "mean")]
    t = _transformer(plan_only=True, comm=Two())
    comp = t.computation(ng.adamw([table, w], shared, lr=0.1), idx, d)
    t.initialize()
    kinds = [s.kind for s in comp.steps]
    assert sorted(kinds) == sorted(["embed", "norm", "norm_grad", "embed_grad", "comm", "comm", "adamw"]) and kinds[-1] == "adamw"
    exchanges = [s for s in comp.steps if s.kind == "comm"]
    assert set(v.buffer for v in comp.steps[-1].gradients) == set(s.arena_buffer for s in exchanges)
    for s in exchanges:
        made = [k for k, x in enumerate(comp.steps) if x.kind != "comm" and s.arena_buffer in [v.buffer for v in x.out_views]]
        assert len(made) == 1 and made[0] < comp.steps.index(s)
    assert sorted(s.reduce_func for s in exchanges) == ["mean", "sum"]


def _gradient_steps(n, gate, which):
    """A computation of the gradients named, over n tokens or rows, and what it has to be called with."""
    V, F, T = _axes(V=40, F=8, T=n)
    rng = np.random.RandomState(n)
    table, idx, d, block = ng.variable([V, F], initial_value=1), ng.placeholder([T]), ng.placeholder([T, F]), ng.placeholder([T, F])
    w = ng.variable([F], initial_value=1)
    e = ng.embedding(table, idx)
    if which is None:
        return ng.embedding_grad(d, e), [idx, d], [rng.randint(0, 40, n), rng.standard_normal((n, 8))]
    g = None if gate is None else ng.variable([dict(F=F, T=T)[k] for k in gate], initial_value=1)
    stream, out = ng.residual_norm(e, block, w, axes=[F], gate=g, post_weight=w)
    found = ng.residual_norm_grad(out, d_out=d)
    return [found[k] for k in which], [idx, d, block], [rng.randint(0, 40, n)] + [rng.standard_normal((n, 8)) for _ in range(2)]


LAUNCHES = [(1, None, None, 1), (256, None, None, 1), (257, None, None, 2), (9, None, ("residual", "block"), 1), (9, None, ("weight",), 2),
            (9, None, ("post_weight",), 2), (9, "F", ("gate",), 2), (9, "T", ("gate", "residual"), 1), (9, "TF", ("gate",), 1)]


@pytest.mark.parametrize("n,gate,which,launches", LAUNCHES)
def test_launches_of_gradients(n, gate, which, launches):
    op, args, _ = _gradient_steps(n, gate, which)
    t = _transformer(plan_only=True)
    comp = t.computation(op, *args)
    t.initialize()
    assert [s.launches for s in comp.steps if s.kind in ("embed_grad", "norm_grad")] == [launches]


# ---- on the device -------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("flex", [False, True])
def test_embedding_and_its_gradient(flex):
    V, F, T, B = _axes(V=37, F=12, T=20, B=3)
    rng = np.random.RandomState(0)
    w, idx = rng.standard_normal((37, 12)).astype(np.float32), rng.randint(0, 37, (3, 20))
    delta = rng.standard_normal((12, 3, 20)).astype(np.float32)
    table, x = ng.variable([V, F], initial_value=w), ng.placeholder([B, T])
    d = ng.placeholder([F, B, T])                       # (as another layer lays it out)
    e = ng.embedding(table, x, scale=3.0, pad_idx=5)
    t = _transformer(flex=flex)
    comp = t.computation([e, ng.embedding_grad(d, e)], x, d)
    for recorded in (False, True):
        out, grad = comp(idx, delta)
        want = np.zeros((37, 12))
        rows = delta.transpose(1, 2, 0).reshape(-1, 12).astype(np.float64)
        keep = idx.reshape(-1) != 5
        np.add.at(want, idx.reshape(-1)[keep], rows[keep] * 3)
        if flex:
            # operands and results off by a step of their tensor at most (host values are cut off, not rounded; an
            # exponent leaves a tensor's largest at a quarter of the range or more), sums of at most 12 rows
            step = lambda a: np.abs(a).max() * 2.0 ** -13  # noqa: E731
            # a result is held with the exponent that its first values have been given: greater ones later are cut off
            # at its 32767 steps
            if not recorded:
                limits = [fx.MANT_MAX * fx.scale_of(fx.fit_dec(np.abs(a).max())) for a in (out, grad)]
            looked_up, want = [np.clip(a, -r, r) for a, r in zip((w[idx] * 3, want), limits)]
            assert np.abs(out - looked_up).max() <= 3 * step(w) + step(out)
            assert np.abs(grad - want).max() <= 3 * 12 * step(delta) + step(grad)
        else:
            assert np.array_equal(out, w[idx] * np.float32(3))
            np.testing.assert_allclose(grad, want, atol=15 * 2.0 ** -24 * np.abs(rows).max() * 36)
        idx, delta = rng.randint(0, 37, (3, 20)), rng.standard_normal((12, 3, 20)).astype(np.float32)
        if not recorded:
            comp.capture()
    t.close()


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [None, "F", "BT", "BTF", "FTB"])
def test_residual_norm_and_its_gradients(gate):
    """Operands in the orders in which they come: rows of a wider tensor, features first."""
    F, T, B = _axes(F=40, T=9, B=4)
    wide = ng.make_axis(100, name="F")
    rng = np.random.RandomState(1)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    lengths, ax = dict(F=40, T=9, B=4), dict(F=F, T=T, B=B)
    res, blk, d_out, d_stream = f(40, 4, 9), f(4, 9, 100), f(4, 9, 40), f(4, 9, 40)
    pre, post = 1 + 0.2 * f(40), 1 + 0.2 * f(40)
    gv = None if gate is None else f(*[lengths[c] for c in gate])
    r, b, do, ds = ng.placeholder([F, B, T]), ng.placeholder([B, T, wide]), ng.placeholder([B, T, F]), ng.placeholder([B, T, F])
    u = ng.cast_axes(ng.tensor_slice(b, [slice(None), slice(None), slice(60, 100)]), [B, T, F])
    g = None if gate is None else ng.placeholder([ax[c] for c in gate])
    w, p = ng.variable([F], initial_value=pre), ng.variable([F], initial_value=post)
    stream, out = ng.residual_norm(r, u, w, axes=[F], post_weight=p, gate=g, residual_scale=0.5, eps=1e-5)
    grads = ng.residual_norm_grad(out, do, ds)
    names = list(grads)
    t = _transformer()
    comp = t.computation([stream, out] + [grads[k] for k in names], *([r, b, do, ds] + ([] if g is None else [g])))
    feed = [res, blk, d_out, d_stream] + ([] if g is None else [gv])
    rows = lambda a, order: a.transpose([order.index(c) for c in "BTF"]).reshape(36, 40)  # noqa: E731
    order = "".join(a.name for a in stream.axes)
    g2 = None if gate is None else gv.reshape(1, 40) if gate == "F" else gv.reshape(36, 1) if gate == "BT" else rows(gv, gate)
    c = (rows(res, "FBT"), blk[:, :, 60:].reshape(36, 40), g2, post, pre, 0.5, 1e-5)
    want, size = no.forward(*c)
    back, back_size = no.backward(want["stream"], want["stream_rstd"], d_out.reshape(36, 40), d_stream.reshape(36, 40), c[1], want["block_rstd"], g2,
                                  post, pre, 0.5)
    key = dict(residual="residual", block="block", gate="gate", post_weight="post", weight="pre")
    for recorded in (False, True):
        got = comp(*feed)
        for v, k in zip(got[:2], ("stream", "out")):
            assert np.all(np.abs(rows(v, order) - want[k]) <= 40 * 2.0 ** -24 * size[k])
        for v, k in zip(got[2:], names):
            v = rows(v, order) if v.ndim == 3 else v.reshape(back[key[k]].shape)
            # (the stream and its reciprocal deviation that the gradients read are those of the pass before, rounded)
            assert np.all(np.abs(v - back[key[k]]) <= 200 * 2.0 ** -24 * back_size[key[k]]), k
        if not recorded:
            comp.capture()
    t.close()


@pytest.mark.gpu
def test_rms_norm_and_only_some_gradients():
    F, T = _axes(F=33, T=7)
    rng = np.random.RandomState(2)
    x, d, wv = rng.standard_normal((7, 33)).astype(np.float32), rng.standard_normal((7, 33)).astype(np.float32), np.ones(33, np.float32)
    xp, dp, w = ng.placeholder([T, F]), ng.placeholder([T, F]), ng.variable([F], initial_value=wv)
    y = ng.rms_norm(xp, w, axes=[F])
    grads = ng.residual_norm_grad(y, d_out=dp)
    assert set(grads) == {"residual", "weight"}
    t = _transformer()
    both = t.computation([y, grads["residual"], grads["weight"]], xp, dp)
    one = t.computation(grads["weight"], xp, dp)
    got = both(x, d)
    want, _ = no.forward(x, pre=wv)
    back, size = no.backward(x, want["stream_rstd"], d, pre=wv)
    np.testing.assert_allclose(got[0], want["out"], rtol=1e-5, atol=1e-6)
    for v, k in zip(got[1:], ("residual", "pre")):
        assert np.all(np.abs(v - back[k]) <= 100 * 2.0 ** -24 * size[k])
    assert np.array_equal(one(x, d), got[2])
    t.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_steps(bits):
    """Bit for bit, a learning rate and a scale that change from call to call, recorded or not; readers of the variable
    before and behind the step see its old and its new value; the moments can be read and set."""
    A, B = _axes(A=300, B=7)
    rng = np.random.RandomState(3)
    v1, v2 = rng.standard_normal((300, 7)).astype(np.float32), rng.standard_normal(7).astype(np.float32)
    w1, w2 = ng.variable([A, B], initial_value=v1), ng.variable([B], initial_value=v2)
    g1, g2, lr, scale = ng.placeholder([B, A]), ng.placeholder([B]), ng.placeholder([]), ng.placeholder([])
    before = ng.sum(w2, out_axes=[]) + 0.0
    step = ng.adamw([w1, w2], [g1, g2 * 2.0], lr=lr, weight_decay=0.1, no_decay=[w2], state_bits=bits, grad_scale=scale, seed=9)
    behind = ng.sum(w2, out_axes=[]) + 1.0
    t = _transformer()
    comp = t.computation([before, step, ng.sequential([step, behind])], g1, g2, lr, scale)
    state = {k: (np.zeros(n, np.float32),) * 2 if bits == 32 else
             (np.zeros(n, np.uint8),) * 2 + (np.zeros(-(-n // 256), np.float32),) * 2 for k, n in ((0, 2100), (1, 7))}
    values = [v1.reshape(-1), v2]
    for k in range(4):
        a, b = (rng.standard_normal((7, 300)) * 0.1).astype(np.float32), rng.standard_normal(7).astype(np.float32)
        rate, factor = float(np.float32(0.01 * (k + 1))), float(np.float32(0.5 ** k))
        old = values[1].copy()
        got = comp(a, b, rate, factor)
        h = (rate, 0.9, 0.999, 1e-8, 0.1)
        values[0], state[0] = ao.step(values[0], np.ascontiguousarray(a.T).reshape(-1), state[0], k + 1, h, 1.0, factor, 9, 0)
        values[1], state[1] = ao.step(values[1], b * np.float32(2), state[1], k + 1, h, 0.0, factor, 9, 2304)
        assert abs(float(got[0]) - old.sum(dtype=np.float64)) < 1e-5 and float(got[1].reshape(-1)[0]) == k + 1
        assert abs(float(got[2]) - 1 - values[1].sum(dtype=np.float64)) < 1e-5
        for w, v in ((w1, values[0]), (w2, values[1])):
            assert np.array_equal(t.device_tensor(w).get(None).reshape(-1), v)
        for s, want in zip(step.states, (state[0], state[1])):
            for x, y in zip(s, want):
                held = np.ascontiguousarray(t.device_tensor(x).get(None)).reshape(-1)
                held = held.view(y.dtype)[:y.size]
                assert np.array_equal(held, y)
        if k == 1:
            comp.capture()
        if k == 2:                                       # kept and put back, as a checkpoint does
            kept = [[np.array(t.device_tensor(x).get(None)) for x in s] for s in step.states]
            for s, held in zip(step.states, kept):
                for x, v in zip(s, held):
                    t.device_tensor(x)[...] = np.zeros_like(v)
                    t.device_tensor(x)[...] = v
    t.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_gradients_that_are_variables(bits):
    A, B = _axes(A=3000, B=70)
    rng = np.random.RandomState(4)
    values = [rng.standard_normal(210000).astype(np.float32) for _ in range(2)]
    x, y = [ng.variable([A, B], initial_value=v.reshape(3000, 70)) for v in values]
    r = ng.variable([], initial_value=0.125)
    step = ng.adamw([x, y, r], [y, x, ng.tensor_slice(x, [1, 2])], lr=r, weight_decay=0.0, state_bits=bits)
    t = _transformer()
    comp = t.computation(step)
    values.append(np.array([0.125], np.float32))
    state = [(np.zeros(v.size, np.float32),) * 2 if bits == 32 else
             (np.zeros(v.size, np.uint8),) * 2 + (np.zeros(-(-v.size // 256), np.float32),) * 2 for v in values]
    for k in range(4):
        comp()
        h = (float(values[2][0]), 0.9, 0.999, 1e-8, 0.0)
        found, at = [], 0
        for v, g, s in zip(values, (values[1], values[0], values[0][72:73]), state):
            found.append(ao.step(v, g, s, k + 1, h, 1.0, 1.0, 0, at))
            at += -(-v.size // 256) * 256
        values, state = [f[0] for f in found], [f[1] for f in found]
        for op, v in zip((x, y, r), values):
            assert np.array_equal(np.asarray(t.device_tensor(op).get(None)).reshape(-1), v)
        if k == 1:
            comp.capture()
    t.close()


def _language_model(n_tokens, vocab, features, layers, bits, lr):
    """A residual network over tokens -- lookup, blocks of a matrix and tanh between norms, an output layer, softmax
    cross-entropy -- with all gradients and an AdamW step."""
    V, F, T = _axes(V=vocab, F=features, T=n_tokens)
    G = ng.make_axis(features, name="G")
    r = np.random.RandomState(0)
    f = lambda s, *n: (r.standard_normal(n) * s).astype(np.float32)  # noqa: E731
    idx, target = ng.placeholder([T]), ng.placeholder([T, V])
    table = ng.variable([V, F], initial_value=f(0.3, vocab, features), name="table")
    head = ng.variable([F, V], initial_value=f(0.2, features, vocab), name="head")
    mats = [ng.variable([F, G], initial_value=f(0.2, features, features), name="mat%d" % k) for k in range(layers)]
    norms = [ng.variable([F], initial_value=1 + f(0.1, features), name="norm%d" % k) for k in range(layers + 1)]
    gates = [ng.variable([F], initial_value=0.5 + f(0.1, features), name="gate%d" % k) for k in range(layers)]
    posts = [ng.variable([F], initial_value=1 + f(0.1, features), name="post%d" % k) for k in range(layers)]
    e = ng.embedding(table, idx, scale=2.0, pad_idx=0)
    out, stream, edges, acts = ng.rms_norm(e, norms[0], axes=[F]), e, [], []
    first = out
    for k in range(layers):
        a = ng.tanh(ng.dot(out, mats[k]))                        # [T, G]
        acts.append((out, a))
        stream, out = ng.residual_norm(stream, ng.cast_axes(a, [T, F]), norms[k + 1], axes=[F], post_weight=posts[k], gate=gates[k], residual_scale=0.9)
        edges.append(out)
    z = ng.dot(out, head)
    ex = ng.exp(z - ng.max(z, reduction_axes=[V]))
    p = ex / ng.sum(ex, reduction_axes=[V])
    loss = ng.sum(ng.negative(ng.sum(target * ng.log(p), reduction_axes=[V])), out_axes=[]) * (1.0 / n_tokens)
    dz = (p - target) * (1.0 / n_tokens)
    grads = {head: ng.dot(out, dz)}
    d_out, d_stream = ng.dot(dz, head), None
    for k in reversed(range(layers)):
        g = ng.residual_norm_grad(edges[k], d_out, d_stream)
        grads.update({norms[k + 1]: g["weight"], posts[k]: g["post_weight"], gates[k]: g["gate"]})
        x, a = acts[k]
        da = ng.cast_axes(g["block"], [T, G]) * (1.0 - a * a)
        grads[mats[k]] = ng.dot(x, da)
        d_out, d_stream = ng.dot(da, mats[k]), g["residual"]
    g = ng.residual_norm_grad(first, d_out, d_stream)
    grads[norms[0]] = g["weight"]
    grads[table] = ng.embedding_grad(g["residual"], e)
    variables = [table, head] + mats + norms + gates + posts
    step = ng.adamw(variables, [grads[v] for v in variables], lr=lr, no_decay=norms + gates + posts, state_bits=bits)
    return dict(idx=idx, target=target, loss=loss, step=step, variables=variables, grads=grads, stream=stream)


def _same_in_torch(values, idx, target, layers):
    """The loss and gradients in 64 bits."""
    import torch
    v = {k: torch.tensor(x, dtype=torch.float64, requires_grad=True) for k, x in values.items()}
    rms = lambda x, w: x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6) * w  # noqa: E731
    i = torch.tensor(idx)
    rows = torch.where((i == 0)[:, None], v["table"].detach()[i], v["table"][i])
    stream = rows * 2
    out = rms(stream, v["norm0"])
    for k in range(layers):
        a = torch.tanh(out @ v["mat%d" % k])
        stream = 0.9 * stream + v["gate%d" % k] * rms(a, v["post%d" % k])
        out = rms(stream, v["norm%d" % (k + 1)])
    loss = -(torch.tensor(target, dtype=torch.float64) * torch.log_softmax(out @ v["head"], 1)).sum(1).mean()
    loss.backward()
    return float(loss.detach()), {k: x.grad.numpy() for k, x in v.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_of_them_all(bits):
    """Lookup, norms, products, AdamW in one computation, step by step and recorded: the loss and every gradient against
    64 bits at the weights of the call, the weights bit for bit from these gradients."""
    T, V, F, L = 60, 41, 24, 2
    m = _language_model(T, V, F, L, bits, 0.01)
    t = _transformer()
    comp = t.computation([m["loss"]] + [m["grads"][v] for v in m["variables"]] + [m["step"]], m["idx"], m["target"])
    t.initialize()
    rng = np.random.RandomState(5)
    states, counters, at = [], [], 0
    for v in m["variables"]:
        n = v.axes.size
        states.append((np.zeros(n, np.float32),) * 2 if bits == 32 else (np.zeros(n, np.uint8),) * 2 + (np.zeros(-(-n // 256), np.float32),) * 2)
        counters.append(at)
        at += -(-n // 256) * 256
    read = lambda v: np.array(t.device_tensor(v).get(None))  # noqa: E731
    for k in range(5):
        idx = rng.randint(0, V, T)
        target = np.eye(V, dtype=np.float32)[rng.randint(0, V, T)]
        values = {v.name: read(v) for v in m["variables"]}
        got = comp(idx.astype(np.float32), target)
        loss, grads = _same_in_torch(values, idx, target, L)
        assert abs(float(got[0]) - loss) < 1e-4 * abs(loss)
        assert float(got[-1].reshape(-1)[0]) == k + 1
        for j, v in enumerate(m["variables"]):
            g = np.asarray(got[1 + j], np.float32)
            want = grads[v.name]
            # products of 24 to 60 terms one behind the other through seven layers, tanh and exp in fp32: some hundred
            # roundings of 2^-24 of what the terms add up to, which for these values is about ten times the largest
            assert np.abs(g.reshape(want.shape) - want).max() <= 500 * 2.0 ** -24 * 10 * np.abs(want).max(), v.name
            hyper = (0.01, 0.9, 0.999, 1e-8, 0.01)
            p, states[j] = ao.step(values[v.name].reshape(-1), g.reshape(-1), states[j], k + 1, hyper, float(m["step"].decayed[j]), 1.0, 0, counters[j])
            assert np.array_equal(read(v).reshape(-1), p), v.name
        if k == 1:
            comp.capture()
    t.close()


@pytest.mark.gpu
def test_the_norms_gradients_are_given_the_status_of_their_transformer(monkeypatch):
    """A wait that runs out in them is an error of the call, as in the other kernels with bounded waits."""
    from ngraph_python_b200 import lib
    F, T = _axes(F=12, T=7)
    x, d, w = ng.placeholder([T, F]), ng.placeholder([T, F]), ng.variable([F], initial_value=1)
    t = _transformer()
    comp = t.computation(ng.residual_norm_grad(ng.rms_norm(x, w, axes=[F]), d_out=d)["residual"], x, d)
    raw, seen = lib.raw(), []

    class Watched(object):
        def __getattr__(self, name):
            return getattr(raw, name)

        def b2_norm_bprop(self, a, grads, *rest):
            seen.append(grads._obj.status)
            return raw.b2_norm_bprop(a, grads, *rest)
    monkeypatch.setattr(lib, "raw", lambda: Watched())
    v = np.ones((7, 12), np.float32)
    comp(v, v)
    assert seen == [t._status.data_ptr()]
    # the word that such a wait sets
    t._status.fill_(1)
    with pytest.raises(lib.B200Error, match="wait ran out"):
        comp(v, v)
    comp(v, v)
    t.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n,gate,which,launches", LAUNCHES)
def test_launches_are_counted_as_they_are(n, gate, which, launches):
    """Nodes of a recording of the step alone."""
    import ctypes
    import torch
    op, args, values = _gradient_steps(n, gate, which)
    t = _transformer()
    comp = t.computation(op, *args)
    comp(*values)
    step, = [s for s in comp.steps if s.kind in ("embed_grad", "norm_grad")]
    graph, nodes, before = torch.cuda.CUDAGraph(keep_graph=True), ctypes.c_size_t(), t.kernel_launches
    with torch.cuda.graph(graph):
        t._launch_step(step)
    assert ctypes.CDLL("libcuda.so.1").cuGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
    assert nodes.value == launches == step.launches == t.kernel_launches - before
    del graph
    t.close()
