"""Rotation and norms of heads and the step of orthogonalised updates as ops of a graph, each against numpy and together in a
training step, step by step and recorded."""
import numpy as np
import pytest

import ngraph_python_b200 as ng
from oracle import adamw_oracle as ao
from oracle import flex_oracle as fx
from oracle import heads_oracle as ho
from oracle import muon_oracle as mo

ngt = ng.transformers
HALF = 2.0 ** -24


def _transformer(**kw):
    return ngt.make_transformer_factory("b200", **kw)()


def _axes(**lengths):
    return [ng.make_axis(n, name=k) for k, n in lengths.items()]


# ---- construction ------------------------------------------------------------------------------------
def test_axes_and_refusals_of_the_ops():
    T, B, H, K, D, V = _axes(T=5, B=3, H=4, K=2, D=8, V=11)
    q, k, at, odd = ng.placeholder([B, T, H, D]), ng.placeholder([K, B, T, D]), ng.placeholder([B, T]), ng.placeholder([T, V])
    w = ng.variable([D], initial_value=1)
    r = ng.Rotation(at, pairs="neighbours", rotary_dim=4)
    y = ng.rotary(k, r, heads=K, features=D)
    assert y.axes == ng.make_axes([B, T, K, D]) and y.place == (15, 1) and y.rotary_dim == 4
    assert ng.rotary(ng.placeholder([T, D]), ng.Rotation(T), heads=None, features=D).axes == ng.make_axes([T, D])
    assert ng.rotary(q, ng.Rotation(T), heads=[H], features=[D]).place == (5, 1) and ng.rotary(q, ng.Rotation(B), heads=H, features=D).place == (3, 5)
    assert ng.rotary_grad(ng.placeholder([D, K, T, B]), y).inverse
    one, two = ng.head_norm([q, k], [w, None], heads=[H, K], features=D, rotation=r)
    assert one.axes == ng.make_axes([B, T, H, D]) and two.axes == ng.make_axes([B, T, K, D])
    g = ng.head_norm_grad([one, two], [one, two])
    assert [x.axes for x in g["x"]] == [one.axes, two.axes] and g["weight"][0].axes == w.axes and g["weight"][1] is None
    m, s = ng.variable([T, V], initial_value=0), ng.variable([H, V, T], initial_value=0)
    step = ng.muon([m, s], [odd, s], lr=0.1, no_decay=[m], scale="rms")
    assert step.shapes == [(1, 5, 11), (4, 11, 5)] and step.decayed == [False, True] and step.scales == [0.2 * 11 ** 0.5] * 2
    assert ng.muon([m, s], [odd, s], lr=0.1).scales == [1.0, (11 / 5) ** 0.5]
    rotation = lambda **kw: (lambda: ng.Rotation(at, **kw))  # noqa: E731
    for build in (rotation(pairs="thirds"), rotation(scaling="other"), rotation(base=0.0), rotation(factor=-1.0), rotation(low=4.0, high=4.0), rotation(amplitude=float("nan")),
                  lambda: ng.rotary(q, at, heads=H, features=D), lambda: ng.rotary(q, ng.Rotation(at, rotary_dim=3), heads=H, features=D),
                  lambda: ng.rotary(q, ng.Rotation(at, rotary_dim=10), heads=H, features=D), lambda: ng.rotary(q, r, heads=K, features=D),
                  lambda: ng.rotary(q, r, heads=D, features=D), lambda: ng.rotary(q, r, heads=H, features=[H, D]), lambda: ng.rotary(q, r, heads=H, features=V),
                  lambda: ng.rotary(q, ng.Rotation(odd), heads=H, features=D), lambda: ng.rotary(q, ng.Rotation(V), heads=H, features=D),
                  lambda: ng.rotary(ng.placeholder([B, V, T, D]), r, heads=None, features=D), lambda: ng.rotary_grad(q, q), lambda: ng.rotary_grad(q, y),
                  lambda: ng.head_norm([q], [w, w], heads=[H], features=D), lambda: ng.head_norm([q, k], [w, w], heads=[H], features=D),
                  lambda: ng.head_norm([q, odd], [None, None], heads=[H, None], features=D), lambda: ng.head_norm([q], [at], heads=[H], features=D),
                  lambda: ng.head_norm([q], [w], heads=[H], features=D, eps=-1.0), lambda: ng.head_norm([q], [w], heads=[H], features=D, rotation=at),
                  lambda: ng.head_norm([q, ng.placeholder([T, K, D])], [w, w], heads=[H, K], features=D),
                  lambda: ng.head_norm([ng.placeholder([T, ng.make_axis(1025, name="D")])], [None], heads=[None], features=ng.make_axis(1025, name="D")),
                  lambda: ng.head_norm_grad([one], [one, two]), lambda: ng.head_norm_grad([one, one], one), lambda: ng.head_norm_grad([one, two], y),
                  lambda: ng.muon([m], [], lr=0.1), lambda: ng.muon([m, m], [odd, odd], lr=0.1), lambda: ng.muon([w], [w], lr=0.1), lambda: ng.muon([y], [y], lr=0.1),
                  lambda: ng.muon([m], [at], lr=0.1), lambda: ng.muon([m], [odd], lr=odd), lambda: ng.muon([m], [odd], lr=0.1, momentum=1.0),
                  lambda: ng.muon([m], [odd], lr=0.1, iterations=0), lambda: ng.muon([m], [odd], lr=0.1, iterations=33), lambda: ng.muon([m], [odd], lr=0.1, scale="other"),
                  lambda: ng.muon([m], [odd], lr=0.1, no_decay=[s]), lambda: ng.muon([m], [odd], lr=0.1, coefficients=(1.0, float("inf"), 0.0))):
        with pytest.raises(ValueError):
            build()


def test_flex_transformers_refuse_norms_and_muon():
    T, D = _axes(T=4, D=8)
    x, m = ng.placeholder([T, D]), ng.variable([T, D], initial_value=1)
    for op in (ng.head_norm([x], [None], heads=[None], features=D)[0], ng.muon([m], [x], lr=0.1)):
        t = _transformer(flex=True, plan_only=True)
        t.computation(op, x)
        with pytest.raises(ValueError, match="not flex16"):
            t.initialize()


def _product(T, H, K, D, wide):
    """Queries and keys as they lie in the rows of one product, with other heads between and behind them."""
    both = ng.make_axis(H.length + K.length + 3, name="C")
    x = ng.placeholder([T, both, D])
    part = lambda a, b, ax: ng.cast_axes(ng.tensor_slice(x, [slice(None), slice(a, b), slice(None)]), [T, ax, D])  # noqa: E731
    return x, part(1, 1 + H.length, H), part(2 + H.length, 2 + H.length + K.length, K)


def test_steps_of_a_plan():
    """One step each, and no copy of operands that lie as they should -- heads among others of a product among them."""
    T, H, K, D = _axes(T=6, H=4, K=2, D=8)
    x, q, k = _product(T, H, K, D, 3)
    w, m = ng.variable([D], initial_value=1), ng.variable([H, D], initial_value=1)
    out = ng.head_norm([q, k], [w, w], heads=[H, K], features=D, rotation=ng.Rotation(T))
    g = ng.head_norm_grad(out, out)
    turned = ng.rotary(q, ng.Rotation(T), heads=H, features=D)
    back = ng.rotary_grad(turned, turned)
    t = _transformer(plan_only=True)
    comp = t.computation([turned, back] + out + g["x"] + g["weight"] + [ng.muon([m], [m * 2.0], lr=0.1)], x)
    t.initialize()
    assert sorted(s.kind for s in comp.steps if s.kind != "ew") == ["head_norm", "head_norm_grad", "muon", "rotary", "rotary"]
    assert {s.kind: s.launches for s in comp.steps if s.kind.startswith("head_norm")} == {"head_norm": 1, "head_norm_grad": 2}
    t = _transformer(plan_only=True)
    y = ng.placeholder([D, H, T])
    comp = t.computation(ng.rotary(y, ng.Rotation(T), heads=H, features=D), y)
    t.initialize()
    assert [s.kind for s in comp.steps] == ["dimshuffle", "rotary"]
    # heads before rows lie as they should
    t = _transformer(plan_only=True)
    y = ng.placeholder([H, T, D])
    comp = t.computation(ng.rotary(y, ng.Rotation(T), heads=H, features=D), y)
    t.initialize()
    assert [s.kind for s in comp.steps] == ["rotary"]


def test_muon_of_gradients_that_are_variables_of_the_step_are_copied_first():
    A, B = _axes(A=5, B=4)
    x, y, g = ng.variable([A, B], initial_value=1), ng.variable([A, B], initial_value=2), ng.placeholder([A, B])
    for op, copies in ((ng.muon([x, y], [y, x], lr=0.1), 2), (ng.muon([x, y], [g, x], lr=0.1), 1), (ng.muon([x], [y], lr=0.1), 0)):
        t = _transformer(plan_only=True)
        comp = t.computation(op, g)
        t.initialize()
        assert [s.kind for s in comp.steps] == ["dimshuffle"] * copies + ["muon"]


# ---- on the device -------------------------------------------------------------------------------------
def _far(got, want, size, steps):
    assert np.all(np.abs(np.asarray(got, np.float64) - want) <= steps * HALF * size), np.max(np.abs(got - want) / (HALF * size + 1e-30))


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("order", ["BTHD", "HTBD", "DTHB"])
@pytest.mark.parametrize("given", ["BT", "T", "axis"])
def test_rotary_and_its_gradient(pairs, order, given):
    """Whatever the order of the axes, positions for every row, shared by sequences, or the place along an axis."""
    lengths = dict(B=3, T=7, H=2, D=12)
    ax = {k: ng.make_axis(n, name=k) for k, n in lengths.items()}
    rng = np.random.RandomState(1)
    shape = lambda s: tuple(lengths[c] for c in s)  # noqa: E731
    v, d = rng.standard_normal(shape(order)).astype(np.float32), rng.standard_normal(shape("HDBT")).astype(np.float32)
    p = rng.randint(0, 5000, shape(given)) if given != "axis" else np.arange(7)
    x, delta, at = ng.placeholder([ax[c] for c in order]), ng.placeholder([ax[c] for c in "HDBT"]), ng.placeholder([ax[c] for c in (given if given != "axis" else "T")])
    r = ng.Rotation(ax["T"] if given == "axis" else at, rotary_dim=8, pairs=pairs, base=500.0, scaling="linear", factor=2.0, amplitude=1.5)
    rows = "".join(c for c in order if c in "BT")
    if given == "BT" and rows == "TB":
        pass                                            # (positions are laid out as the rows are)
    y = ng.rotary(x, r, heads=ax["H"], features=ax["D"])
    assert "".join(a.name for a in y.axes) == rows + "HD"
    t = _transformer()
    comp = t.computation([y, ng.rotary_grad(delta, y)], *([x, delta] + ([at] if given != "axis" else [])))
    for recorded in (False, True):
        out, grad = comp(*([v, d] + ([p] if given != "axis" else [])))
        flat = lambda a, o: np.transpose(a, [o.index(c) for c in rows + "HD"]).reshape(-1, 2, 12)  # noqa: E731
        every = np.broadcast_to(np.transpose(p, [given.index(c) for c in rows])[...] if given == "BT" else p.reshape([7 if c == "T" else 1 for c in rows]), shape(rows)).reshape(-1)
        angle = every[:, None] * ho.frequencies(8, base=500.0, scaling="linear", factor=2.0)
        for got, value, inverse in ((out, flat(v, order), False), (grad, flat(d, "HDBT"), True)):
            want, size = ho.rotate(value, angle, 8, pairs == "neighbours", 1.5, inverse)
            _far(got.reshape(-1, 2, 12), want, size, 6)
        v, d = v[..., ::-1].copy(), d[::-1].copy()
        if given != "axis":
            p = p + 3
        if not recorded:
            comp.capture()
    t.close()


@pytest.mark.gpu
@pytest.mark.parametrize("given", [True, False])
def test_rotary_in_flex16(given):
    """Operands are cut to a step of their tensor, a result is off by half a step of its own on top (values that outgrow the
    exponent of the first call are cut off)."""
    T, H, D = _axes(T=9, H=3, D=16)
    rng = np.random.RandomState(2)
    v, p = rng.standard_normal((9, 3, 16)).astype(np.float32), rng.randint(0, 900, 9)
    x, at = ng.placeholder([T, H, D]), ng.placeholder([T])
    y = ng.rotary(x, ng.Rotation(at if given else T), heads=H, features=D)
    t = _transformer(flex=True)
    comp = t.computation([y, ng.rotary_grad(y, y)], *([x, at] if given else [x]))
    for recorded in (False, True):
        out, back = comp(*([v, p] if given else [v]))
        angle = (p if given else np.arange(9))[:, None] * ho.frequencies(16)
        want, size = ho.rotate(v, angle, 16, False)
        step = lambda a: np.abs(a).max() * 2.0 ** -13  # noqa: E731
        if not recorded:
            limit = fx.MANT_MAX * fx.scale_of(fx.fit_dec(np.abs(out).max()))
        assert np.abs(out - np.clip(want, -limit, limit)).max() <= 3 * step(v) + step(out)
        assert np.abs(back - ho.rotate(out, angle, 16, False, 1.0, True)[0]).max() <= 3 * step(out) + step(back)
        v = v[::-1].copy()
        if not recorded:
            comp.capture()
    t.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rotated", [True, False])
@pytest.mark.parametrize("weights", [(True, True), (True, False)])
def test_head_norm_and_its_gradients(rotated, weights):
    """Heads among those of one product; with weights, and without one, and only some gradients read."""
    T, H, K, D = _axes(T=21, H=4, K=2, D=10)
    rng = np.random.RandomState(4)
    x, q, k = _product(T, H, K, D, 3)
    w = [ng.variable([D], initial_value=(1 + 0.3 * rng.standard_normal(10)).astype(np.float32)) if has else None for has in weights]
    at, dq, dk = ng.placeholder([T]), ng.placeholder([T, H, D]), ng.placeholder([K, T, D])
    r = ng.Rotation(at, rotary_dim=6, amplitude=1.25) if rotated else None
    out = ng.head_norm([q, k], w, heads=[H, K], features=D, rotation=r, eps=1e-5)
    g = ng.head_norm_grad([dq, dk], out)
    some = [x for x in g["x"] + g["weight"] if x is not None]
    t = _transformer()
    comp = t.computation(out + some, *([x, dq, dk] + ([at] if rotated else [])))
    alone = t.computation(g["weight"][0], *([x, dq, dk] + ([at] if rotated else [])))
    for recorded in (False, True):
        v, d0, d1, p = rng.standard_normal((21, 9, 10)).astype(np.float32), rng.standard_normal((21, 4, 10)).astype(np.float32), \
            rng.standard_normal((2, 21, 10)).astype(np.float32), rng.randint(0, 9999, 21)
        args = [v, d0, d1] + ([p] if rotated else [])
        got = comp(*args)
        assert np.array_equal(alone(*args), got[4])
        angle = p[:, None] * ho.frequencies(6)
        d = 6 if rotated else 0
        for i, (part, delta) in enumerate(((v[:, 1:5], d0), (v[:, 6:8], d1.transpose(1, 0, 2)))):
            weight = None if w[i] is None else np.asarray(t.device_tensor(w[i]).get(None))
            want, rstd, size = ho.forward(part, weight, 1e-5, angle, d, False, 1.25)
            _far(got[i], want, size, 30)
            dx, dw, dx_size, dw_size = ho.backward(delta, part, weight, rstd, angle, d, False, 1.25)
            # (the stored deviation is off by up to eight halves of a step, which enters three times)
            _far(got[2 + i], dx, dx_size, 70)
            if weight is not None:
                _far(got[4 + i], dw, dw_size, 200)
        if not recorded:
            comp.capture()
    t.close()


def _moved(before, mean, grad, lr, scale, decay=0.0, mu=0.95, grad_scale=1.0):
    """(param, mean) after a step in 64 bits, and how far the param may be off in the 2-norm."""
    x, mean = mo.update(grad, mean, mu, scale=grad_scale)
    want = before * (1 - lr * decay) - lr * scale * mo.orthogonal(x)[0]
    far = lr * scale * (mo.reach(x) + 8 * HALF * 4 ** 5) + 4 * HALF * np.sqrt(np.sum(before ** 2) + np.sum(want ** 2))
    return want, mean, far


@pytest.mark.gpu
def test_muon_steps():
    """A matrix, a stack of them and a tall one, whose gradient another layer lays out; a rate and a scale that change from call to
    call, recorded or not; readers before and behind the step; the means are persistent."""
    A, B, S = _axes(A=40, B=70, S=3)
    rng = np.random.RandomState(3)
    f = lambda *s: (rng.standard_normal(s) * 0.1).astype(np.float32)  # noqa: E731
    values = [f(40, 70), f(3, 40, 70), f(70, 40)]
    ws = [ng.variable([A, B], initial_value=values[0]), ng.variable([S, A, B], initial_value=values[1]), ng.variable([B, A], initial_value=values[2])]
    g = ng.placeholder([A, B]), ng.placeholder([A, S, B]), ng.placeholder([B, A])
    lr, scale = ng.placeholder([]), ng.placeholder([])
    before = ng.sum(ws[0], out_axes=[]) + 0.0
    step = ng.muon(ws, [g[0], g[1] * 2.0, g[2]], lr=lr, weight_decay=0.1, no_decay=[ws[1]], grad_scale=scale)
    behind = ng.sum(ws[0], out_axes=[]) + 1.0
    t = _transformer()
    comp = t.computation([before, step, ng.sequential([step, behind])], *(list(g) + [lr, scale]))
    means = [np.zeros_like(v) for v in values]
    for k in range(4):
        grads = [f(40, 70), f(40, 3, 70), f(70, 40)]
        rate, factor = float(np.float32(0.02 * (k + 1))), 0.5 ** k
        old = values[0].sum(dtype=np.float64)
        got = comp(*(grads + [rate, factor]))
        assert abs(float(got[0]) - old) < 1e-4 and float(got[1].reshape(-1)[0]) == k + 1
        for i, (w, gr) in enumerate(zip(ws, (grads[0], grads[1].transpose(1, 0, 2) * 2, grads[2]))):
            held, mean = np.array(t.device_tensor(w).get(None)), np.array(t.device_tensor(step.states[i]).get(None))
            for j in range(3 if i == 1 else 1):
                at = (j,) if i == 1 else ()
                want, m, far = _moved(values[i][at], means[i][at], gr[at], rate, (70 / 40) ** 0.5 if i == 2 else 1.0, 0.0 if i == 1 else 0.1, grad_scale=factor)
                assert np.sqrt(np.sum((held[at] - want) ** 2)) <= far
                assert np.all(np.abs(mean[at] - m) <= 6 * HALF * (np.abs(means[i][at]) + np.abs(gr[at])))
            values[i], means[i] = held, mean
        assert abs(float(got[2]) - 1 - values[0].sum(dtype=np.float64)) < 1e-4
        if k == 1:
            comp.capture()
    t.close()


def _language_model(n_tokens, vocab, features, heads, dim, lr):
    """One block over tokens: lookup, norm, one product for queries and keys, their norms with the rotation, an elementwise meeting of
    every query head with its key head, a product back, the norm behind, an output layer and softmax cross-entropy, all gradients; the
    matrices by orthogonalised updates, the rest by AdamW."""
    T, V, F, H, K, J, D = _axes(T=n_tokens, V=vocab, F=features, H=heads, K=1, J=heads + 1, D=dim)
    r = np.random.RandomState(0)
    f = lambda s, *n: (r.standard_normal(n) * s).astype(np.float32)  # noqa: E731
    idx, target, at = ng.placeholder([T]), ng.placeholder([T, V]), ng.placeholder([T])
    v = dict(table=ng.variable([V, F], initial_value=f(0.5, vocab, features), name="table"), head=ng.variable([F, V], initial_value=f(0.3, features, vocab), name="head"),
             qk=ng.variable([F, J, D], initial_value=f(0.4, features, heads + 1, dim), name="qk"), back=ng.variable([H, D, F], initial_value=f(0.4, heads, dim, features), name="back"),
             wq=ng.variable([D], initial_value=1 + f(0.1, dim), name="wq"), wk=ng.variable([D], initial_value=1 + f(0.1, dim), name="wk"),
             w0=ng.variable([F], initial_value=1 + f(0.1, features), name="w0"), w1=ng.variable([F], initial_value=1 + f(0.1, features), name="w1"))
    e = ng.embedding(v["table"], idx, scale=2.0)
    x = ng.rms_norm(e, v["w0"], axes=[F])
    both = ng.dot(x, v["qk"])                                           # [T, J, D]
    q = ng.cast_axes(ng.tensor_slice(both, [slice(None), slice(0, heads), slice(None)]), [T, H, D])
    k = ng.cast_axes(ng.tensor_slice(both, [slice(None), slice(heads, heads + 1), slice(None)]), [T, K, D])
    rotation = ng.Rotation(at, rotary_dim=dim // 2)
    nq, nk = ng.head_norm([q, k], [v["wq"], v["wk"]], heads=[H, K], features=D, rotation=rotation)
    key = ng.tensor_slice(nk, [slice(None), 0, slice(None)])            # [T, D]
    a = ng.tanh(nq * key)                                               # [T, H, D]
    block = ng.dot(a, v["back"])                                        # [T, F]
    stream, out = ng.residual_norm(e, block, v["w1"], axes=[F])
    z = ng.dot(out, v["head"])
    ex = ng.exp(z - ng.max(z, reduction_axes=[V]))
    p = ex / ng.sum(ex, reduction_axes=[V])
    loss = ng.sum(ng.negative(ng.sum(target * ng.log(p), reduction_axes=[V])), out_axes=[]) * (1.0 / n_tokens)
    dz = (p - target) * (1.0 / n_tokens)
    g = ng.residual_norm_grad(out, ng.dot(dz, v["head"]))
    grads = dict(head=ng.dot(out, dz), w1=g["weight"], back=ng.dot(a, g["block"]))
    da = ng.dot(g["block"], v["back"]) * (1.0 - a * a)                  # [T, H, D]
    d_key = ng.sum(da * nq, reduction_axes=[H])
    heads_grads = ng.head_norm_grad([da * key, ng.cast_axes(ng.broadcast(d_key, [T, K, D]), [T, K, D])], [nq, nk])
    grads.update(wq=heads_grads["weight"][0], wk=heads_grads["weight"][1])
    dq, dk = heads_grads["x"]
    wq_part, wk_part = [ng.dot(x, d) for d in (dq, dk)]                 # [F, H, D], [F, K, D]
    return dict(T=T, idx=idx, target=target, at=at, loss=loss, v=v, grads=grads, parts=(wq_part, wk_part), dq=dq, dk=dk, e=e, x=x, g=g, H=H, K=K, J=J, F=F, D=D, lr=lr)


@pytest.mark.gpu
def test_a_training_step_of_them_all():
    """The loss and every gradient against 64 bits at the weights of the call, the weights from these gradients: matrices where the
    orthogonalised step takes them, the others bit for bit as AdamW does; step by step and recorded."""
    import torch
    n, vocab, features, heads, dim = 30, 23, 16, 3, 8
    T, V, F, H, K, D = _axes(T=n, V=vocab, F=features, H=heads, K=1, D=dim)
    m = _language_model(n, vocab, features, heads, dim, 0.02)
    v, grads = m["v"], dict(m["grads"])
    # the gradient of the joint matrix and of the lookup: both parts side by side
    q_w = ng.cast_axes(ng.tensor_slice(v["qk"], [slice(None), slice(0, heads), slice(None)]), [m["F"], m["H"], m["D"]])
    k_w = ng.cast_axes(ng.tensor_slice(v["qk"], [slice(None), slice(heads, heads + 1), slice(None)]), [m["F"], m["K"], m["D"]])
    joint = ng.variable([m["F"], m["J"], m["D"]], initial_value=0, name="joint")
    fill = ng.sequential([ng.assign(ng.tensor_slice(joint, [slice(None), slice(0, heads), slice(None)]), ng.cast_axes(m["parts"][0], [m["F"], ng.make_axis(heads, name="J"), m["D"]])),
                          ng.assign(ng.tensor_slice(joint, [slice(None), slice(heads, heads + 1), slice(None)]), ng.cast_axes(m["parts"][1], [m["F"], ng.make_axis(1, name="J"), m["D"]])), joint])
    d_x = ng.dot(m["dq"], q_w) + ng.dot(m["dk"], k_w)                   # [T, F]
    first = ng.residual_norm_grad(m["x"], d_x, m["g"]["residual"])
    grads.update(qk=fill, w0=first["weight"], table=ng.embedding_grad(first["residual"], m["e"]))
    matrices, others = ["back", "qk"], ["table", "head", "wq", "wk", "w0", "w1"]
    muon = ng.muon([v[k] for k in matrices], [grads[k] for k in matrices], lr=0.02, scale="rms")
    adamw = ng.adamw([v[k] for k in others], [grads[k] for k in others], lr=0.01, weight_decay=0.0)
    t = _transformer()
    names = sorted(v)
    comp = t.computation([m["loss"]] + [grads[k] for k in names] + [muon, adamw], m["idx"], m["target"], m["at"])
    t.initialize()
    rng = np.random.RandomState(5)
    read = lambda op: np.array(t.device_tensor(op).get(None))  # noqa: E731
    states = {k: (np.zeros(v[k].axes.size, np.float32),) * 2 for k in others}
    counters, total = {}, 0
    for k in others:
        counters[k] = total
        total += -(-v[k].axes.size // 256) * 256
    means = {k: np.zeros(v[k].axes.lengths) for k in matrices}
    for step in range(4):
        idx, at, target = rng.randint(0, vocab, n), rng.randint(0, 500, n), np.eye(vocab, dtype=np.float32)[rng.randint(0, vocab, n)]
        held = {k: read(v[k]) for k in names}
        got = comp(idx.astype(np.float32), target, at.astype(np.float32))
        w = {k: torch.tensor(x, dtype=torch.float64, requires_grad=True) for k, x in held.items()}
        rms = lambda x: x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)  # noqa: E731
        angle = torch.tensor(at[:, None] * ho.frequencies(dim // 2))[:, None]
        c, s, h = torch.cos(angle), torch.sin(angle), dim // 4

        def turned(y):
            a, b = y[..., :h], y[..., h:2 * h]
            return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * h:]], -1)
        e = w["table"][torch.tensor(idx)] * 2
        both = torch.einsum("tf,fjd->tjd", rms(e) * w["w0"], w["qk"])
        q, k = turned(rms(both[:, :heads]) * w["wq"]), turned(rms(both[:, heads:]) * w["wk"])
        block = torch.einsum("thd,hdf->tf", torch.tanh(q * k), w["back"])
        out = rms(e + block) * w["w1"]
        loss = -(torch.tensor(target, dtype=torch.float64) * torch.log_softmax(out @ w["head"], 1)).sum(1).mean()
        loss.backward()
        assert abs(float(got[0]) - float(loss.detach())) < 1e-4 * abs(float(loss.detach()))
        for k, x in zip(names, got[1:]):
            want = w[k].grad.numpy()
            # as in the training step of the other operators: some hundred roundings of what the terms add up to, which here is
            # about ten times the largest gradient
            assert np.abs(np.asarray(x).reshape(want.shape) - want).max() <= 500 * HALF * 10 * np.abs(want).max(), k
        for k in others:
            x = np.asarray(got[1 + names.index(k)], np.float32).reshape(-1)
            p, states[k] = ao.step(held[k].reshape(-1), x, states[k], step + 1, (0.01, 0.9, 0.999, 1e-8, 0.0), 1.0, 1.0, 0, counters[k])
            assert np.array_equal(read(v[k]).reshape(-1), p), k
        for k in matrices:
            x, now = np.asarray(got[1 + names.index(k)], np.float32).reshape(held[k].shape), read(v[k])
            for j in range(held[k].shape[0]):
                want, mean, far = _moved(held[k][j], means[k][j], x[j], 0.02, 0.2 * max(x[j].shape) ** 0.5)
                assert np.sqrt(np.sum((now[j] - want) ** 2)) <= far, k
                means[k][j] = mean
        if step == 1:
            comp.capture()
    t.close()


@pytest.mark.gpu
def test_one_operand_twice_and_gradients_that_are_broadcast():
    """Both tensors of heads are one placeholder with one weight, the results' gradients are the same for all rows or for all heads and
    features, and one position is everybody's."""
    T, H, D = _axes(T=333, H=3, D=16)
    rng = np.random.RandomState(8)
    x, at, by_feature, by_row = ng.placeholder([T, H, D]), ng.placeholder([]), ng.placeholder([D]), ng.placeholder([T])
    weight = (1 + 0.3 * rng.standard_normal(16)).astype(np.float32)
    w = ng.variable([D], initial_value=weight)
    out = ng.head_norm([x, x], [w, w], heads=[H, H], features=D, rotation=ng.Rotation(at))
    g = ng.head_norm_grad([ng.broadcast(by_feature, [T, H, D]), ng.broadcast(by_row, [T, H, D])], out)
    t = _transformer()
    comp = t.computation(out + g["x"] + g["weight"], x, at, by_feature, by_row)
    for recorded in (False, True):
        v, d0, d1, p = [rng.standard_normal(s).astype(np.float32) for s in ((333, 3, 16), (16,), (333,))] + [int(rng.randint(9999))]
        got = comp(v, p, d0, d1)
        angle = p * ho.frequencies(16)[None, :] + np.zeros((333, 1))
        want, rstd, size = ho.forward(v, weight, 1e-6, angle, 16, False, 1.0)
        for i, delta in enumerate((np.broadcast_to(d0, v.shape), np.broadcast_to(d1[:, None, None], v.shape))):
            _far(got[i], want, size, 30)
            dx, dw, dx_size, dw_size = ho.backward(delta, v, weight, rstd, angle, 16, False, 1.0)
            _far(got[2 + i], dx, dx_size, 70)
            _far(got[4 + i], dw, dw_size, 200)
        if not recorded:
            comp.capture()
    t.close()


@pytest.mark.gpu
def test_one_gradient_of_two_matrices_and_one_step_of_two_computations():
    """Two variables follow one gradient; computations that share the step, one of them recorded, go on from one another's state."""
    A, B = _axes(A=100, B=150)
    rng = np.random.RandomState(9)
    start = [(rng.standard_normal((100, 150)) * 0.1).astype(np.float32) for _ in range(2)]
    g = ng.placeholder([A, B])
    ws = [ng.variable([A, B], initial_value=s) for s in start]
    step = ng.muon(ws, [g, g], lr=0.05, nesterov=True)
    t = _transformer()
    one, two = t.computation(step, g), t.computation([step, ng.sum(g, out_axes=[])], g)
    values, mean = [s.copy() for s in start], np.zeros((100, 150))
    for k in range(4):
        grad = rng.standard_normal((100, 150)).astype(np.float32)
        got = two(grad)[0] if k % 2 else one(grad)
        assert float(np.asarray(got).reshape(-1)[0]) == k + 1
        for i, w in enumerate(ws):
            want, m, far = _moved(values[i], mean, grad, 0.05, 1.0)
            held = np.array(t.device_tensor(w).get(None))
            assert np.sqrt(np.sum((held - want) ** 2)) <= far
            values[i] = held
        mean = np.array(t.device_tensor(step.states[0]).get(None))
        assert np.array_equal(mean, np.array(t.device_tensor(step.states[1]).get(None)))
        if k == 1:
            two.capture()
    t.close()
