"""Rotation of heads by position and norms of heads with the rotation in the same pass, through the C ABI, against 64 bits.

How far a value may be off: a cosine or sine by three halves of a step of one -- its angle, at most an eighth of a turn, is
rounded to fp32 (0.8 of half a step of one), the function is good to a step (of values below one: half of a step of one is its
whole step), the amplitude rounds once -- and the products and the sum of a rotation round twice more.  That is 5 halves of a
step of |u| + |v| for a rotated pair (u, v); six are granted.  Norms add a mean of squares, as in the norms between blocks."""
import ctypes

import numpy as np
import pytest

from oracle import heads_oracle as ho

HALF = 2.0 ** -24
KINDS = {"f32": (0, np.float32), "i32": (1, np.int32), "i64": (2, np.int64), "i16": (3, np.int16)}


class _Heads(object):
    """A device tensor [rows][heads][D] with strides of its own, in a sea of marks."""
    MARK = -77

    def __init__(self, value, row=None, head=None, offset=0):
        import torch
        value = np.ascontiguousarray(value)
        R, H, D = value.shape
        self.head = D if head is None else head
        self.row = max(H, 1) * self.head if row is None else row
        self.shape, self.offset = value.shape, offset
        size = offset + max(R - 1, 0) * self.row + max(H - 1, 0) * self.head + D + 8
        self.all = torch.full((size,), self.MARK, dtype=torch.from_numpy(value).dtype, device="cuda")
        self.t = torch.as_strided(self.all, value.shape, (self.row, self.head, 1), offset)
        self.t.copy_(torch.from_numpy(value))
        self.ptr = self.all.data_ptr() + self.all.element_size() * offset

    def intact(self):
        import torch
        seen = torch.ones_like(self.all, dtype=torch.bool)
        torch.as_strided(seen, self.shape, (self.row, self.head, 1), self.offset).fill_(False)
        return bool((self.all[seen] == self.MARK).all())

    def get(self):
        return self.t.cpu().numpy()


def _strides(lay, R, H, D):
    """(row, head, offset) of a layout: dense, one head after another with a gap, heads before rows, off 16 bytes."""
    return {"dense": (H * D, D, 0), "apart": (H * (D + 4) + 12, D + 4, 4), "odd": (H * (D + 3) + 5, D + 3, 1), "heads first": (D, R * D, 0),
            "fused": ((H + 6) * D, D, 2 * D)}[lay]


def _args(R, D, rotary, interleaved, turns=None, positions=None, kind="i64", count=None, group=1, amplitude=1.0, inverse=0, eps=1e-6, parts=2):
    from ngraph_python_b200 import lib
    a = lib.HeadsArgs()
    a.rows, a.head_dim, a.rotary_dim, a.interleaved, a.inverse = R, D, rotary, int(interleaved), inverse
    a.turns = None if turns is None else turns.data_ptr()
    a.positions = None if positions is None else positions.data_ptr()
    a.position_kind, a.position_count, a.position_group = KINDS[kind][0], R if count is None else count, group
    a.amplitude, a.eps, a.parts = amplitude, eps, parts
    return a


def _turns(rotary, **kw):
    from ngraph_python_b200 import lib
    t = lib.rotary_turns(rotary, **kw)
    return t, t.cuda()


def _data(R, H, D, seed=0):
    rng = np.random.RandomState(seed + R + 7 * H + D)
    return rng.standard_normal((R, H, D)).astype(np.float32)


def _positions(R, kind, seed=0, most=100000):
    import torch
    p = np.random.RandomState(seed + R).randint(0, most, R)
    return p, torch.from_numpy(p.astype(KINDS[kind][1])).cuda()


def _ok(got, want, size, steps, what=""):
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= steps * HALF * size), (what, float(np.max(err / (HALF * np.maximum(size, 1e-30)))))


SIZES = [(1, 1, 0, 1, 0), (1, 32, 8, 128, 128), (16, 4, 1, 64, 64), (3, 3, 2, 2, 2), (33, 5, 5, 77, 76), (7, 12, 4, 80, 40), (130, 2, 2, 96, 48),
         (5, 3, 1, 256, 256), (2, 2, 2, 1024, 1024), (3, 1, 1, 1001, 500), (700, 8, 2, 16, 8), (9, 40, 8, 128, 2), (11, 3, 3, 24, 10), (4, 2, 1, 520, 260),
         (3000, 3, 1, 32, 32), (6, 2, 2, 192, 128), (5, 7, 1, 66, 64), (2500, 8, 8, 8, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R,q,k,D,rotary", SIZES)
@pytest.mark.parametrize("lay", ["dense", "apart", "odd", "heads first"])
def test_rotation(R, q, k, D, rotary, interleaved, lay):
    import torch
    from ngraph_python_b200 import lib
    turns, on = _turns(rotary, scaling="parts", factor=4.0, original=512.0)
    kind = ("i64", "i32", "f32")[(R + D) % 3]
    p, positions = _positions(R, kind)
    angle = ho.angles(p, turns.numpy())
    for inverse in (0, 1):
        a = _args(R, D, rotary, interleaved, on, positions, kind, amplitude=1.25, inverse=inverse)
        x = [_data(R, h, D, s) for s, h in ((0, q), (1, k))]
        ins = [_Heads(v, *_strides(lay, R, v.shape[1], D)) for v in x]
        outs = [_Heads(np.zeros_like(v), *_strides(lay, R, v.shape[1], D)) for v in x]
        for i in range(2):
            s, o = ins[i], outs[i]
            a.part[i].heads, a.part[i].x, a.part[i].out = x[i].shape[1], s.ptr, o.ptr
            a.part[i].x_row, a.part[i].x_head, a.part[i].out_row, a.part[i].out_head = s.row, s.head, o.row, o.head
        lib.check(lib.raw().b2_rotary(ctypes.byref(a), 0, None, None, None, 0, None))
        torch.cuda.synchronize()
        for v, s, o in zip(x, ins, outs):
            want, size = ho.rotate(v, angle, rotary, interleaved, 1.25, bool(inverse))
            assert o.intact() and s.intact() and np.array_equal(s.get(), v)
            _ok(o.get(), want, size, 6)
            assert np.array_equal(o.get()[..., rotary:], v[..., rotary:])


def _rotate_one(x, rotary, interleaved, positions=None, kind="i64", count=None, group=1, turns=None, in_place=False, rows=None):
    import torch
    from ngraph_python_b200 import lib
    R, H, D = x.shape
    turns, on = _turns(rotary) if turns is None else (turns, turns.cuda())
    a = _args(R, D, rotary, interleaved, on, positions, kind, count, group, parts=1)
    s = _Heads(x)
    o = s if in_place else _Heads(np.zeros_like(x))
    a.part[0].heads, a.part[0].x, a.part[0].out = H, s.ptr, o.ptr
    a.part[0].x_row = a.part[0].out_row = s.row
    a.part[0].x_head = a.part[0].out_head = s.head
    lib.check(lib.raw().b2_rotary(ctypes.byref(a), 0, None, None, None, 0, None))
    torch.cuda.synchronize()
    return o.get()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rotary", [(64, 64), (21, 12)])
def test_far_positions(interleaved, D, rotary):
    """Whole numbers of 64 bits, negative ones among them: the angles are exact but for the frequencies' own rounding."""
    import torch
    turns, _ = _turns(rotary)
    p = np.array([0, 1, -1, 1 << 20, (1 << 24) + 1, -(1 << 31), (1 << 40) + 12345, (1 << 62) + 1, -(1 << 63), (1 << 63) - 1])
    x = _data(len(p), 3, D)
    got = _rotate_one(x, rotary, interleaved, torch.from_numpy(p).cuda(), turns=turns)
    want, size = ho.rotate(x, ho.angles(p, turns.numpy()), rotary, interleaved)
    _ok(got, want, size, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rotary", [(64, 32), (21, 12)])
def test_positions_that_are_not_numbers(D, rotary):
    """The rotated features of such a row are NaN, the others and other rows are what they are."""
    import torch
    p = torch.tensor([3.0, float("nan"), float("inf"), -float("inf"), 1e19, 2.4, 5.5], device="cuda")
    x = _data(7, 2, D)
    got = _rotate_one(x, rotary, False, p, "f32")
    assert np.isnan(got[1:5, :, :rotary]).all() and np.array_equal(got[..., rotary:], x[..., rotary:])
    turns, _ = _turns(rotary)
    want, size = ho.rotate(x[[0, 5, 6]], ho.angles([3, 2, 6], turns.numpy()), rotary, False)
    _ok(got[[0, 5, 6]], want, size, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rotary", [(32, 32), (21, 12)])
@pytest.mark.parametrize("count,group", [(4, 1), (4, 3), (1, 1), (100, 5), (12, 1), (3, 4)])
def test_positions_that_rows_share(D, rotary, count, group):
    """Row r reads position (r / group) % count, or is at it where there are none."""
    x = _data(12, 2, D)
    turns, _ = _turns(rotary)
    p, positions = _positions(count, "i32")
    index = np.arange(12) // group % count
    for given, at in ((positions, p[index]), (None, index)):
        got = _rotate_one(x, rotary, True, given, "i32", count, group, turns)
        want, size = ho.rotate(x, ho.angles(at, turns.numpy()), rotary, True)
        _ok(got, want, size, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rotary", [(128, 128), (64, 32), (77, 40)])
def test_rotation_in_place(interleaved, D, rotary):
    x = _data(50, 5, D)
    p, positions = _positions(50, "i64")
    assert np.array_equal(_rotate_one(x, rotary, interleaved, positions, in_place=True), _rotate_one(x, rotary, interleaved, positions))


@pytest.mark.parametrize("d", [2, 16, 40, 128])
@pytest.mark.parametrize("scaling", ["none", "linear", "base", "parts"])
def test_frequencies(d, scaling):
    """In 2^-64 of a turn; 2^-50 relative for the powers and products in 64 bits of their making."""
    from ngraph_python_b200 import lib
    kw = dict(base=500.0, scaling=scaling, factor=8.0, original=300.0, low=1.0, high=20.0)
    got = lib.rotary_turns(d, **kw).numpy().astype(np.uint64).astype(np.float64) / 2.0 ** 64
    want = ho.frequencies(d, **kw) / (2 * np.pi) % 1.0
    assert np.all(np.abs(got - want) <= want * 2.0 ** -48 + 2.0 ** -64)


def test_frequencies_of_more_than_a_turn():
    """A base below one: whole turns are left out."""
    from ngraph_python_b200 import lib
    got = lib.rotary_turns(8, base=0.01).numpy().astype(np.uint64).astype(np.float64) / 2.0 ** 64
    want = ho.frequencies(8, base=0.01) / (2 * np.pi)
    assert want[-1] > 1 and np.all(np.abs(got - want % 1.0) <= want * 2.0 ** -48)


# ---- flex16 ----------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R,H,D,rotary,lay", [(5, 3, 64, 64, "dense"), (40, 2, 33, 20, "dense"), (7, 4, 128, 64, "apart"), (9, 2, 16, 16, "odd"), (900, 3, 32, 32, "heads first")])
@pytest.mark.parametrize("kind", ["i16", "f32"])
def test_rotation_in_flex16(R, H, D, rotary, lay, interleaved, kind):
    """Mantissas are the nearest to a value that is off by six halves of a step of fp32: one step away only where the exact
    value is so near the middle between two of them.  The largest one is the statistic, or what a measuring launch leaves."""
    import torch
    from ngraph_python_b200 import lib
    rng = np.random.RandomState(R)
    x = rng.randint(-30000, 30001, (R, H, D)).astype(np.int16)
    dec = (12, 3, 11)                   # of the operand, the positions, the result
    scales = torch.tensor([[2.0 ** -d, 2.0 ** d] for d in dec], device="cuda")
    stats = torch.zeros((3,), dtype=torch.int32, device="cuda")
    probe = torch.zeros((1,), dtype=torch.int64, device="cuda")
    p = rng.randint(0, 3000, R)
    positions = torch.from_numpy((p * 8).astype(np.int16) if kind == "i16" else p.astype(np.float32)).cuda()
    turns, on = _turns(rotary)
    s, o = _Heads(x, *_strides(lay, R, H, D)), _Heads(np.zeros_like(x), *_strides(lay, R, H, D))
    a = _args(R, D, rotary, interleaved, on, positions, kind, parts=1)
    a.slot_positions = 1
    q = a.part[0]
    q.heads, q.x, q.out, q.x_row, q.x_head, q.out_row, q.out_head, q.slot_x, q.slot_out = H, s.ptr, o.ptr, s.row, s.head, o.row, o.head, 0, 2
    call = lambda probing: lib.check(lib.raw().b2_rotary(ctypes.byref(a), 1, scales.data_ptr(), stats.data_ptr(), probe.data_ptr(), probing, None))  # noqa: E731
    call(1)
    torch.cuda.synchronize()
    assert not o.get().any() and not stats.cpu().numpy().any()
    value, size = ho.rotate(x.astype(np.float64) * 2.0 ** -dec[0], ho.angles(p, turns.numpy()), rotary, interleaved)
    found = probe.cpu().numpy().astype(np.uint32).view(np.float32)[0]
    assert abs(found - np.abs(value).max()) <= 6 * HALF * size.max()
    call(0)
    torch.cuda.synchronize()
    want = np.clip(value * 2.0 ** dec[2], -32768, 32767)
    got = o.get().astype(np.float64)
    assert o.intact() and np.all(np.abs(got - want) <= 0.5 + 6 * HALF * size * 2.0 ** dec[2])
    assert stats.cpu().tolist() == [0, 0, int(np.abs(got).max())]


# ---- norms -----------------------------------------------------------------------------------------------
def _norm(R, q, k, D, rotary, interleaved, lay="dense", weights=(True, True), in_place=False, keep=True, backward=False, seed=0, x=None, amplitude=0.75,
          eps=1e-6, wanted=(True, True)):
    """Runs fprop, or fprop and bprop; ([out, rstd] or [d_x, d_weight] of both tensors, what they were made from)."""
    import torch
    from ngraph_python_b200 import lib
    turns, on = _turns(rotary)
    kind = ("i64", "i32", "f32")[(R + D) % 3]
    p, positions = _positions(max(R, 1), kind)
    a = _args(R, D, rotary, interleaved, on if rotary else None, positions if rotary else None, kind, max(R, 1), amplitude=amplitude, eps=eps)
    x = [_data(R, h, D, seed + s) * np.float32(2) for s, h in ((0, q), (1, k))] if x is None else x
    w = [(1 + 0.3 * _data(1, 1, D, seed + s)[0, 0]).astype(np.float32) if has else None for s, has in ((2, weights[0]), (3, weights[1]))]
    wd = [None if v is None else torch.from_numpy(v).cuda() for v in w]
    ins = [_Heads(v, *_strides(lay, R, v.shape[1], D)) for v in x]
    outs = ins if in_place else [_Heads(np.zeros_like(v), *_strides(lay, R, v.shape[1], D)) for v in x]
    rstd = [torch.full((max(R * v.shape[1], 1),), -7.0, device="cuda") for v in x]
    for i in range(2):
        s, o = ins[i], outs[i]
        c = a.part[i]
        c.heads, c.x, c.out, c.x_row, c.x_head, c.out_row, c.out_head = x[i].shape[1], s.ptr, o.ptr, s.row, s.head, o.row, o.head
        c.weight, c.rstd = None if wd[i] is None else wd[i].data_ptr(), rstd[i].data_ptr() if keep else None
    lib.check(lib.raw().b2_heads_fprop(ctypes.byref(a), None))
    torch.cuda.synchronize()
    info = dict(x=x, w=w, angle=ho.angles(p[:R], turns.numpy()), args=a, rotary=rotary, interleaved=interleaved, amplitude=amplitude, eps=eps,
                hold=(on, positions, wd, ins, outs, rstd))
    assert all(o.intact() for o in outs + ins)
    found = [(o.get(), r[:R * v.shape[1]].cpu().numpy().reshape(R, v.shape[1])) for o, r, v in zip(outs, rstd, x)]
    if not backward:
        return found, info
    d = [_data(R, v.shape[1], D, seed + 9 + i) for i, v in enumerate(x)]
    ds = [_Heads(v, *_strides(lay, R, v.shape[1], D)) for v in d]
    dx = ds if in_place else [_Heads(np.zeros_like(v), *_strides(lay, R, v.shape[1], D)) for v in d]
    dw = [torch.full((D + 2,), -7.0, device="cuda") for _ in x]
    g = lib.HeadsGrads()
    for i in range(2):
        c = g.part[i]
        c.d_out, c.d_out_row, c.d_out_head = ds[i].ptr, ds[i].row, ds[i].head
        c.d_x, c.d_x_row, c.d_x_head = dx[i].ptr if wanted[0] else None, dx[i].row, dx[i].head
        c.d_weight = dw[i].data_ptr() + 4 if w[i] is not None and wanted[1] else None
    n = lib.heads_bprop_scratch_bytes(a)
    scratch = torch.full((n + 64,), 255, dtype=torch.uint8, device="cuda")
    call = lambda st=None: lib.check(lib.raw().b2_heads_bprop(ctypes.byref(a), ctypes.byref(g), scratch.data_ptr(), n, st))  # noqa: E731
    call()
    torch.cuda.synchronize()
    assert all(v.intact() for v in ds + dx) and scratch[n:].eq(255).all()
    assert all(v[0] == -7 and v[-1] == -7 for v in dw)
    info.update(d=d, rstd=[f[1] for f in found], call=call, grads=g, hold=info["hold"] + (ds, dx, dw, scratch), scratch=scratch, bytes=n)
    return [(o.get(), v[1:-1].cpu().numpy()) for o, v in zip(dx, dw)], info


def _check_norm(found, info, keep=True):
    for (out, rstd), x, w in zip(found, info["x"], info["w"]):
        want, r, size = ho.forward(x, w, info["eps"], info["angle"], info["rotary"], info["interleaved"], info["amplitude"])
        steps = x.shape[2] / 32 + 24
        _ok(out, want, size, steps)
        if keep:
            _ok(rstd, r, r, steps)
        else:
            assert np.all(rstd == -7)


def _check_grads(found, info, weights=True):
    for i, (dx, dw) in enumerate(found):
        x, w = info["x"][i], info["w"][i]
        want, want_w, size, size_w = ho.backward(info["d"][i], x, w, info["rstd"][i], info["angle"], info["rotary"], info["interleaved"], info["amplitude"])
        R, H, D = x.shape
        _ok(dx, want, size, D / 32 + 40, "x")
        if w is not None and weights:
            # the longest chain of additions: what one warp adds, its CTA's warps, and the CTAs' sums by 32 and then 32
            _ok(dw, want_w, size_w, R * H / 100 + 150, "weight")


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R,q,k,D,rotary", SIZES + [(5, 2, 1, 64, 0), (40, 3, 1, 33, 0)])
@pytest.mark.parametrize("lay", ["dense", "odd", "heads first", "fused"])
def test_norm(R, q, k, D, rotary, interleaved, lay):
    _check_norm(*_norm(R, q, k, D, rotary, interleaved, lay))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R,q,k,D,rotary", SIZES + [(5, 2, 1, 64, 0), (40, 3, 1, 33, 0)])
@pytest.mark.parametrize("lay", ["dense", "odd", "heads first", "fused"])
def test_norm_gradients(R, q, k, D, rotary, interleaved, lay):
    _check_grads(*_norm(R, q, k, D, rotary, interleaved, lay, backward=True))


@pytest.mark.gpu
@pytest.mark.parametrize("D,rotary,lay", [(128, 128, "fused"), (64, 32, "dense"), (33, 20, "odd"), (8, 8, "apart")])
@pytest.mark.parametrize("weights", [(True, False), (False, False)])
def test_norm_in_place_and_without_weights(D, rotary, lay, weights):
    _check_norm(*_norm(21, 5, 2, D, rotary, False, lay, weights, in_place=True, keep=False), keep=False)
    found, info = _norm(21, 5, 2, D, rotary, False, lay, weights, backward=True)
    _check_grads(found, info)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rotary", [(128, 64), (33, 20)])
def test_gradients_in_place_and_some_alone(D, rotary):
    full, info = _norm(70, 5, 2, D, rotary, True, backward=True)
    in_place = _norm(70, 5, 2, D, rotary, True, backward=True, in_place=False, wanted=(True, False))[0]
    weights = _norm(70, 5, 2, D, rotary, True, backward=True, wanted=(False, True))[0]
    for f, p, w in zip(full, in_place, weights):
        assert np.array_equal(f[0], p[0]) and np.all(p[1] == -7) and np.array_equal(f[1], w[1]) and not w[0].any()
    # d_x in the place of d_out
    import torch
    for i in range(2):
        c = info["grads"].part[i]
        c.d_x, c.d_x_row, c.d_x_head = c.d_out, c.d_out_row, c.d_out_head
    info["call"]()
    torch.cuda.synchronize()
    for i, ds in enumerate(info["hold"][6]):
        assert np.array_equal(ds.get(), full[i][0])


@pytest.mark.gpu
@pytest.mark.parametrize("R,q,k,D", [(9000, 3, 1, 64), (5000, 1, 1, 40), (20000, 1, 0, 31), (3000, 16, 16, 128), (40000, 1, 1, 8)])
def test_gradients_of_many_rows_are_the_same_bits_in_every_run(R, q, k, D):
    found, info = _norm(R, q, k, D, D // 4 * 2, False, backward=True)
    _check_grads(found, info)
    import torch
    first = [v.clone() for v in info["hold"][8]]
    for _ in range(3):
        info["scratch"].random_(0, 255)
        info["call"]()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, info["hold"][8]))


@pytest.mark.gpu
def test_nothing_to_do():
    """No rows or no heads: nothing is stored but weight gradients, which are zero."""
    for R, q, k in ((0, 3, 1), (4, 0, 0), (4, 2, 0)):
        found, info = _norm(R, q, k, 16, 16, False, backward=True)
        if R == 0 or q == 0:
            assert not any(f[1].any() for f in found)
        else:
            _check_grads(found[:1], info)
            assert not found[1][1].any()
    _rotate_one(np.zeros((0, 3, 16), np.float32), 16, False, count=1)
    _rotate_one(np.zeros((3, 0, 16), np.float32), 16, False)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rotary", [(64, 64), (33, 20)])
def test_heads_of_zeros_infinities_and_nan(D, rotary):
    """A head of zeros gives zeros (its deviation is eps alone); what is not finite stays in its own head."""
    x = [_data(6, 3, D), _data(6, 1, D, 1)]
    x[0][1, 1] = 0.0
    x[0][2, 0, 3] = np.inf
    x[0][4, 2, 1] = np.nan
    x[1][3, 0] = 3e30                   # squares overflow: the head becomes zeros, as x * (1 / inf) says
    found, info = _norm(6, 3, 1, D, rotary, False, x=x, weights=(True, True))
    (out, rstd), (out_k, rstd_k) = found
    assert not out[1, 1].any() and abs(rstd[1, 1] - 1000) < 0.01
    assert rstd[2, 0] == 0 and np.isnan(out[2, 0, 3]) and np.isnan(rstd[4, 2]) and np.isnan(out[4, 2]).all()
    assert rstd_k[3, 0] == 0 and not out_k[3].any()
    good = np.ones((6, 3), bool)
    good[2, 0] = good[4, 2] = False
    want, r, size = ho.forward(np.where(good[..., None], x[0], 1), info["w"][0], 1e-6, info["angle"], rotary, False, 0.75)
    _ok(out[good], want[good], size[good], D / 32 + 24)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(interleaved):
    """Central differences of sum(d * out) in 64 bits, where their own error is far below what is asked for."""
    found, info = _norm(4, 2, 1, 12, 8, interleaved, backward=True)
    rng = np.random.RandomState(3)
    for i in range(2):
        x, w, d = info["x"][i].astype(np.float64), info["w"][i].astype(np.float64), info["d"][i]
        loss = lambda x, w: np.sum(d * ho.forward(x, w, 1e-6, info["angle"], 8, interleaved, 0.75)[0])  # noqa: E731
        for _ in range(5):
            u, h = rng.standard_normal(x.shape), 1e-5
            assert abs((loss(x + h * u, w) - loss(x - h * u, w)) / (2 * h) - np.sum(u * found[i][0])) < 1e-5 * np.sum(np.abs(u * found[i][0])) + 1e-5
            v = rng.standard_normal(w.shape)
            assert abs((loss(x, w + h * v) - loss(x, w - h * v)) / (2 * h) - np.sum(v * found[i][1])) < 1e-5 * np.sum(np.abs(v * found[i][1])) + 1e-5


def test_the_oracles_gradients_against_autograd():
    torch = pytest.importorskip("torch")
    rng = np.random.RandomState(0)
    x, w, d = rng.standard_normal((3, 2, 10)), rng.standard_normal(10), rng.standard_normal((3, 2, 10))
    angle = rng.standard_normal((3, 3)) * 9
    for interleaved in (False, True):
        a, b = ho.places(6, interleaved)
        xt, wt = torch.from_numpy(x).requires_grad_(), torch.from_numpy(w).requires_grad_()
        y = xt * torch.rsqrt(xt.square().mean(2, keepdim=True) + 1e-6) * wt
        c, s = 1.5 * torch.cos(torch.from_numpy(angle))[:, None], 1.5 * torch.sin(torch.from_numpy(angle))[:, None]
        out = y.clone()
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        want, rstd, _ = ho.forward(x, w, 1e-6, angle, 6, interleaved, 1.5)
        assert np.allclose(out.detach().numpy(), want, atol=1e-13)
        gx, gw = torch.autograd.grad(out, (xt, wt), torch.from_numpy(d))
        dx, dw, _, _ = ho.backward(d, x, w, rstd, angle, 6, interleaved, 1.5)
        assert np.allclose(gx.numpy(), dx, atol=1e-12) and np.allclose(gw.numpy(), dw, atol=1e-12)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rotary", [(128, 128), (33, 20)])
def test_recorded_and_replayed_on_two_streams(D, rotary):
    """A recorded forward and backward pass, replayed on new values, and at the same time on another stream with a scratch of its own."""
    import torch
    from ngraph_python_b200 import lib
    runs = [_norm(300, 6, 2, D, rotary, False, backward=True, seed=s) for s in (0, 50)]
    streams, graphs = [torch.cuda.Stream() for _ in runs], []
    for (found, info), st in zip(runs, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            lib.check(lib.raw().b2_heads_fprop(ctypes.byref(info["args"]), st.cuda_stream))
            info["call"](st.cuda_stream)
        graphs.append(graph)
    for _, info in runs:
        for x in info["hold"][3]:
            x.t.mul_(1.5)
        for o in info["hold"][4] + info["hold"][7]:
            o.t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, info in runs:
        info["x"] = [x.get() for x in info["hold"][3]]
        outs, rstd = info["hold"][4], [r.cpu().numpy().reshape(300, -1) for r in info["hold"][5]]
        _check_norm([(o.get(), r) for o, r in zip(outs, rstd)], info)
        info["rstd"] = rstd
        _check_grads([(o.get(), w[1:-1].cpu().numpy()) for o, w in zip(info["hold"][7], info["hold"][8])], info)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [8, 9])
def test_large_offsets(D):
    """Rows and heads that lie more than 2^31 values apart."""
    import torch
    from ngraph_python_b200 import lib
    far = (1 << 31) + 64
    x = torch.empty((far + 2 * D,), device="cuda")
    (turns, on), positions = _turns(8), torch.tensor([5, 9], device="cuda")
    a = _args(2, D, 8, False, on, positions, parts=1)
    value = torch.from_numpy(_data(2, 2, D)).cuda()
    for row, head in ((far, D), (D, far)):
        v = torch.as_strided(x, (2, 2, D), (row, head, 1))
        v.copy_(value)
        p = a.part[0]
        p.heads, p.x, p.out, p.x_row, p.x_head, p.out_row, p.out_head = 2, x.data_ptr(), x.data_ptr(), row, head, row, head
        lib.check(lib.raw().b2_rotary(ctypes.byref(a), 0, None, None, None, 0, None))
        torch.cuda.synchronize()
        want, size = ho.rotate(value.cpu().numpy(), ho.angles([5, 9], turns.numpy()), 8, False)
        _ok(v.cpu().numpy(), want, size, 6)
        lib.check(lib.raw().b2_heads_fprop(ctypes.byref(a), None))


@pytest.mark.gpu
def test_operands_in_page_locked_memory_and_a_result_on_the_host():
    import torch
    from ngraph_python_b200 import lib
    for D, rotary in ((64, 64), (33, 20)):
        found, info = _norm(12, 3, 1, D, rotary, False, backward=True)
        a, g = info["args"], info["grads"]
        keep = []

        def host(h):
            pinned = h.all.cpu().pin_memory()
            keep.append(pinned)
            return pinned.data_ptr() + 4 * h.offset
        for i in range(2):
            a.part[i].x = host(info["hold"][3][i])
            g.part[i].d_out = host(info["hold"][6][i])
            w = info["hold"][2][i].cpu().pin_memory()
            keep.append(w)
            a.part[i].weight = w.data_ptr()
        lib.check(lib.raw().b2_heads_fprop(ctypes.byref(a), None))
        info["call"]()
        torch.cuda.synchronize()
        _check_norm([(o.get(), r.cpu().numpy().reshape(12, -1)) for o, r in zip(info["hold"][4], info["hold"][5])], info)
        _check_grads([(o.get(), w[1:-1].cpu().numpy()) for o, w in zip(info["hold"][7], info["hold"][8])], info)
        was, a.part[0].out = a.part[0].out, keep[0].data_ptr()
        a.part[0].x = info["hold"][3][0].ptr
        assert lib.raw().b2_heads_fprop(ctypes.byref(a), None) != 0 and b"is not device memory" in lib.raw().b2_last_error()
        a.part[0].out, a.part[1].x = was, torch.zeros(4000).data_ptr()
        assert lib.raw().b2_heads_fprop(ctypes.byref(a), None) != 0


# ---- refusals ---------------------------------------------------------------------------------------------
def _fake(**changes):
    """A call whose addresses are only compared: heads of 4 rows, 2 and 1 heads of 8 features."""
    from ngraph_python_b200 import lib
    a = lib.HeadsArgs()
    a.rows, a.head_dim, a.rotary_dim, a.turns, a.amplitude, a.eps, a.parts = 4, 8, 8, 1 << 30, 1.0, 1e-6, 2
    a.positions, a.position_kind, a.position_count, a.position_group = 1 << 31, 2, 4, 1
    for i, h in ((0, 2), (1, 1)):
        p = a.part[i]
        p.heads, p.x, p.out, p.x_row, p.x_head, p.out_row, p.out_head = h, (1 << 20) * (1 + i), (1 << 20) * (5 + i), 8 * h, 8, 8 * h, 8
    for k, v in changes.items():
        *path, last = k.split("__")
        to = a
        for name in path:
            to = to.part[int(name[1:])] if name[0] == "p" and name[1:].isdigit() else getattr(to, name)
        setattr(to, last, v)
    return a


BAD = [dict(rows=-1), dict(head_dim=0), dict(head_dim=1025), dict(rotary_dim=3), dict(rotary_dim=10), dict(rotary_dim=-2), dict(parts=0), dict(parts=3),
       dict(amplitude=float("nan")), dict(eps=-1.0), dict(eps=float("inf")), dict(turns=None), dict(turns=(1 << 30) + 4), dict(position_count=0),
       dict(position_group=0), dict(position_kind=4), dict(position_kind=-1), dict(positions=(1 << 31) + 4), dict(p0__heads=-1), dict(p0__x=(1 << 20) + 2),
       dict(p1__out=(1 << 20) + 1), dict(p0__x=None), dict(p1__out=None), dict(p0__x_row=-8), dict(p0__x_head=-8), dict(p0__x_row=1 << 50),
       dict(p0__out_row=8), dict(p0__out_head=4), dict(p0__out_head=0), dict(p0__out_row=15),
       # results on operands, on one another, and in place with other strides
       dict(p0__out=(1 << 20) + 32), dict(p0__out=1 << 21), dict(p1__out=(1 << 20) * 5), dict(p1__out=(1 << 20) * 5 + 32), dict(p0__out=1 << 31),
       dict(p0__out=(1 << 30) - 32), dict(p0__out=1 << 20, p0__out_row=20)]


@pytest.mark.parametrize("bad", BAD, ids=[" ".join("%s=%s" % i for i in b.items()) for b in BAD])
def test_refusals(bad):
    from ngraph_python_b200 import lib
    a = _fake(**bad)
    assert lib.raw().b2_rotary(ctypes.byref(a), 0, None, None, None, 0, None) == -1
    assert lib.raw().b2_last_error()
    assert lib.raw().b2_heads_fprop(ctypes.byref(a), None) == -1


def test_more_refusals():
    from ngraph_python_b200 import lib
    raw = lib.raw()

    def refused(rc, text):
        assert rc == -1 and text in raw.b2_last_error().decode(), raw.b2_last_error()
    a = _fake()
    rotary = lambda a, flex=0, scales=1 << 33, stats=1 << 34, probe_out=1 << 35, probe=0: raw.b2_rotary(ctypes.byref(a), flex, scales, stats, probe_out, probe, None)  # noqa: E731
    refused(rotary(_fake(p0__weight=1 << 36)), "without a norm")
    refused(rotary(_fake(p1__rstd=1 << 36)), "without a norm")
    refused(rotary(a, flex=1), "one tensor")
    refused(rotary(_fake(parts=1), flex=1, scales=None), "missing exponents")
    refused(rotary(_fake(parts=1), flex=1, stats=None), "missing exponents")
    refused(rotary(_fake(parts=1), flex=1, probe_out=None, probe=1), "missing exponents")
    refused(rotary(_fake(parts=1, p0__slot_x=-1), flex=1), "missing exponents")
    refused(rotary(_fake(parts=1), flex=1, stats=(1 << 34) + 2), "between two addresses")
    refused(rotary(_fake(position_kind=3), scales=None), "exponent")
    refused(rotary(_fake(position_kind=3, slot_positions=-1)), "exponent")
    refused(raw.b2_rotary(None, 0, None, None, None, 0, None), "missing")
    refused(raw.b2_heads_fprop(ctypes.byref(_fake(inverse=1)), None), "turned back")
    refused(raw.b2_heads_fprop(ctypes.byref(_fake(position_kind=3)), None), "flex16 positions")
    refused(raw.b2_heads_fprop(ctypes.byref(_fake(p0__rstd=(1 << 20) * 5)), None), "one place")
    refused(raw.b2_heads_fprop(ctypes.byref(_fake(p0__rstd=(1 << 36) + 2)), None), "between two addresses")
    refused(raw.b2_heads_fprop(ctypes.byref(_fake(p0__weight=(1 << 20) * 5 + 64)), None), "overlaps an operand")
    n = lib.heads_bprop_scratch_bytes(a)

    def bprop(a, scratch=1 << 38, nbytes=n, **changes):
        g = lib.HeadsGrads()
        for i, h in ((0, 2), (1, 1)):
            a.part[i].weight, a.part[i].rstd = (1 << 36) + 4096 * i, (1 << 37) + 4096 * i
            p = g.part[i]
            p.d_out, p.d_x, p.d_weight = (1 << 39) * (1 + i), (1 << 39) * (3 + i), (1 << 39) * (5 + i)
            p.d_out_row = p.d_x_row = 8 * h
            p.d_out_head = p.d_x_head = 8
        for k, v in changes.items():
            setattr(a.part[0] if k in ("weight", "rstd", "x") else g.part[0], k, v)
        return raw.b2_heads_bprop(ctypes.byref(a), ctypes.byref(g), scratch, nbytes, None)
    refused(bprop(_fake(), scratch=None), "scratch")
    refused(bprop(_fake(), nbytes=n - 1), "scratch")
    refused(bprop(_fake(), weight=None), "not there")
    refused(bprop(_fake(), rstd=None), "reads x, rstd")
    refused(bprop(_fake(), x=None), "reads x, rstd")
    refused(bprop(_fake(), d_out=None), "reads x, rstd")
    refused(bprop(_fake(), d_out_row=-1), "strides")
    refused(bprop(_fake(), d_x_row=15), "overlaps itself")
    refused(bprop(_fake(), d_x=(1 << 39) + 2), "between two addresses")
    refused(bprop(_fake(), d_x=(1 << 39) + 32), "overlaps an operand")
    refused(bprop(_fake(), d_x=1 << 39, d_x_row=24), "other strides")
    refused(bprop(_fake(), d_x=1 << 20), "in the place of an operand")
    refused(bprop(_fake(), d_weight=(1 << 39) * 6), "one place")
    refused(bprop(_fake(), d_weight=(1 << 38) + 64), "overlap")
    refused(bprop(_fake(), d_weight=(1 << 37) + 16), "overlaps an operand")
    refused(raw.b2_heads_bprop(ctypes.byref(a), None, 1 << 38, n, None), "missing")
    for bad in (dict(rotary_dim=3), dict(rotary_dim=2000), dict(rotary_dim=-2), dict(base=0.0), dict(base=float("nan")), dict(scaling="linear", factor=0.0),
                dict(scaling="parts", factor=2.0, original=0.0), dict(scaling="parts", factor=2.0, low=3.0, high=3.0)):
        with pytest.raises(lib.B200Error):
            lib.rotary_turns(**dict(dict(rotary_dim=8), **bad))
    with pytest.raises(ValueError):
        lib.rotary_turns(8, scaling="other")


def test_results_among_operands_of_the_same_rows_are_not_refused():
    """Queries and keys in the rows of one product, each in its own place; refused only for want of a device."""
    from ngraph_python_b200 import lib
    row = 32
    a = _fake(p0__x_row=row, p0__out_row=row, p1__x=(1 << 20) + 64, p1__x_row=row, p1__out_row=row, p0__out=1 << 20, p1__out=(1 << 20) + 64)
    rc = lib.raw().b2_rotary(ctypes.byref(a), 0, None, None, None, 0, None)
    assert rc != -1 or b"not device memory" in lib.raw().b2_last_error() or b"cuda" in lib.raw().b2_last_error().lower()
