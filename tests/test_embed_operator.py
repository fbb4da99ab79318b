"""Table lookups with a scale and the table's gradient by sorted tokens, through the C ABI: forward bit for bit,
sums against 64 bits within what additions in fp32 round, flex16 mantissas exactly."""
import ctypes
import math

import numpy as np
import pytest

from oracle import flex_oracle as fx

KINDS = {"f32": 0, "i32": 1, "i64": 2, "flex16": 3}
PLAIN = (None, -1, -1, -1, None, None, 0)


def _tokens(idx, kind):
    import torch
    dtype = {"f32": np.float32, "i32": np.int32, "i64": np.int64, "flex16": np.int16}[kind]
    return torch.from_numpy(np.asarray(idx).astype(dtype)).cuda()


def _off(shape, dtype, offset):
    """A dense device tensor that begins `offset` elements behind a 16-byte boundary."""
    import torch
    n = int(np.prod(shape))
    return torch.zeros((n + 16,), dtype=dtype, device="cuda")[offset:offset + n].view(shape)


def _lookup(table, idx, kind, scale, offset=0):
    import torch
    from ngraph_python_b200 import lib
    V, F = table.shape
    w = _off(table.shape, torch.float32, offset)
    w.copy_(torch.from_numpy(table))
    x = _tokens(idx, kind)
    out = _off((len(idx), F), torch.float32, offset)
    lib.check(lib.raw().b2_embed_fprop(w.data_ptr(), x.data_ptr(), out.data_ptr(), 0, KINDS[kind], V, F, len(idx), scale, *PLAIN, 0))
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _update(delta, idx, kind, V, scale, pad=-1, onto=None, offset=0, scratch=None):
    import torch
    from ngraph_python_b200 import lib
    n, F = delta.shape
    d = _off(delta.shape, torch.float32, offset)
    d.copy_(torch.from_numpy(delta))
    x = _tokens(idx, kind)
    out = _off((V, F), torch.float32, offset)
    out.copy_(torch.full((V, F), 7.0) if onto is None else torch.from_numpy(onto))
    nbytes = lib.embed_update_scratch_bytes(V, F, n)
    if scratch is None:
        scratch = torch.full((nbytes,), 0xA5, dtype=torch.uint8, device="cuda")
    lib.check(lib.raw().b2_embed_update(d.data_ptr(), x.data_ptr(), out.data_ptr(), 0, KINDS[kind], V, F, n, scale, pad, int(onto is not None), *PLAIN,
                                        scratch.data_ptr(), scratch.numel(), 0))
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _sums(delta, idx, V, scale, pad):
    """The sums in 64 bits, what their terms add up to, and how many there are."""
    idx = np.asarray(idx).astype(np.int64)
    keep = (idx >= 0) & (idx < V) & (idx != pad)
    want, size = np.zeros((V, delta.shape[1])), np.zeros((V, delta.shape[1]))
    np.add.at(want, idx[keep], delta[keep].astype(np.float64))
    np.add.at(size, idx[keep], np.abs(delta[keep]).astype(np.float64))
    return want * scale, size * abs(scale), np.bincount(idx[keep], minlength=V)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "i32", "i64"])
@pytest.mark.parametrize("n,F,V,offset", [(1, 1, 1, 0), (1, 64, 9, 0), (7, 300, 11, 0), (5, 33, 40, 0), (600, 512, 1000, 0), (1000, 2048, 50, 0),
                                          (4096, 64, 70000, 0), (900, 256, 33, 1), (30000, 7, 5, 3)])
def test_lookup(kind, n, F, V, offset):
    rng = np.random.RandomState(n + F)
    table = rng.standard_normal((V, F)).astype(np.float32)
    idx = rng.randint(0, V, n)
    scale = np.float32(math.sqrt(F) * 0.7)
    assert np.array_equal(_lookup(table, idx, kind, float(scale), offset), table[idx] * scale)


@pytest.mark.gpu
def test_tokens_that_name_no_row():
    table = np.random.RandomState(0).standard_normal((10, 8)).astype(np.float32)
    for kind, bad in (("f32", [-1, 10, 1e30, -1e30, np.nan, np.inf, -np.inf]), ("i32", [-1, 10, 2 ** 31 - 1, -2 ** 31]),
                      ("i64", [-1, 10, 2 ** 32 + 3, -2 ** 63])):
        idx = np.array(bad + [3], dtype=np.float64 if kind == "f32" else object)
        out = _lookup(table, idx, kind, 2.0)
        assert np.array_equal(out[-1], table[3] * np.float32(2)) and not out[:-1].any()
        delta = np.ones((len(idx), 8), np.float32)
        want = np.zeros((10, 8), np.float32)
        want[3] = 2
        assert np.array_equal(_update(delta, idx, kind, 10, 2.0), want)


@pytest.mark.gpu
@pytest.mark.parametrize("onto", [False, True])
@pytest.mark.parametrize("kind,n,F,V,pad,offset", [
    ("f32", 1, 1, 1, -1, 0), ("f32", 1, 64, 9, -1, 0), ("i64", 33, 4, 1, -1, 0), ("f32", 32, 8, 2, -1, 0), ("i32", 65, 12, 3, 1, 0),
    ("f32", 300, 24, 37, 5, 0), ("i64", 5000, 100, 7, 0, 0), ("f32", 3001, 301, 1009, 3, 0), ("i32", 2000, 516, 149, -1, 0),
    ("i64", 4097, 256, 20000, 0, 1), ("f32", 100003, 8, 257, -1, 0), ("i32", 1000, 1, 1000003, 999999, 0), ("f32", 700, 2052, 300, -1, 0)])
def test_gradient(kind, n, F, V, pad, offset, onto):
    """One rounding an addition and one of the product: (additions + 2) half steps of the sum of the terms' sizes;
    onto a table, one addition more."""
    rng = np.random.RandomState(n + V)
    delta = rng.standard_normal((n, F)).astype(np.float32)
    idx = np.minimum((rng.uniform(1, V + 1, n) ** rng.uniform(0, 1, n)).astype(np.int64) - 1, V - 1).clip(0)
    scale = float(np.float32(1.7))
    old = rng.standard_normal((V, F)).astype(np.float32) if onto else None
    got = _update(delta, idx, kind, V, scale, pad, old, offset)
    want, size, count = _sums(delta, idx, V, scale, pad)
    room = (count[:, None] + 2) * 2.0 ** -24 * size
    if onto:
        untouched = count == 0
        assert np.array_equal(got[untouched], old[untouched])
        want = want + old
        room = room + 2.0 ** -24 * (np.abs(want) + room)
    assert np.all(np.abs(got - want) <= room * 1.001)
    assert np.array_equal(got, _update(delta, idx, kind, V, scale, pad, old, offset))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [31, 32, 33, 64, 65, 1000, 70001])
def test_one_token_throughout(n):
    """A row of many parts beside empty ones, whole numbers: exact."""
    delta = np.random.RandomState(n).randint(-8, 9, (n, 36)).astype(np.float32)
    for V, token in ((1, 0), (200, 149)):
        want = np.zeros((V, 36), np.float32)
        want[token] = delta.sum(0)
        assert np.array_equal(_update(delta, np.full(n, token), "i32", V, 1.0), want)
        assert not _update(delta, np.full(n, token), "i32", V, 1.0, pad=token).any()


@pytest.mark.gpu
def test_sums_are_added_in_the_order_of_the_tokens():
    """Rows of at most 32 tokens: the bits of one addition after another."""
    rng = np.random.RandomState(3)
    delta = (rng.standard_normal((600, 20)) * 10.0 ** rng.randint(-3, 4, (600, 1))).astype(np.float32)
    idx = np.repeat(np.arange(20), 30)
    rng.shuffle(idx)
    want = np.zeros((20, 20), np.float32)
    for t, v in enumerate(idx):
        want[v] = want[v] + delta[t]
    assert np.array_equal(_update(delta, idx, "f32", 20, 1.0), want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [33, 64, 200, 256, 257, 300, 5000])
def test_parts_of_long_rows(n):
    """The bits of parts of 32 tokens added up one after another, whichever kernels a size takes."""
    rng = np.random.RandomState(n)
    delta = (rng.standard_normal((n, 12)) * 10.0 ** rng.randint(-3, 4, (n, 1))).astype(np.float32)
    idx = rng.choice([2, 4], n, p=[0.8, 0.2])
    want = np.zeros((6, 12), np.float32)
    for v in (2, 4):
        rows = delta[idx == v]
        parts = []
        for at in range(0, len(rows), 32):
            part = np.zeros(12, np.float32)
            for r in rows[at:at + 32]:
                part = part + r
            parts.append(part)
        for part in parts:
            want[v] = want[v] + part
    assert np.array_equal(_update(delta, idx, "i32", 6, 1.0), want)
    old = rng.standard_normal((6, 12)).astype(np.float32)
    assert np.array_equal(_update(delta, idx, "i64", 6, 1.0, onto=old), old + want)


@pytest.mark.gpu
def test_no_tokens():
    empty = np.zeros((0, 6), np.float32)
    assert not _update(empty, [], "f32", 5, 1.0).any()
    old = np.random.RandomState(0).standard_normal((5, 6)).astype(np.float32)
    assert np.array_equal(_update(empty, [], "i64", 5, 1.0, onto=old), old)


@pytest.mark.gpu
def test_infinities_reach_their_rows_alone():
    delta = np.ones((40, 8), np.float32)
    delta[3, 2], delta[4, 5], delta[9, 0] = np.inf, np.nan, -np.inf
    idx = np.arange(40) % 10
    got = _update(delta, idx, "f32", 10, 1.0)
    bad = ~np.isfinite(got)
    assert np.array_equal(np.argwhere(bad), [[3, 2], [4, 5], [9, 0]]) and np.all(got[~bad] == 4)


@pytest.mark.gpu
@pytest.mark.parametrize("n,F,V,offset", [(1, 1, 1, 0), (300, 24, 37, 0), (3001, 301, 1009, 0), (900, 512, 30, 0), (500, 64, 9, 1),
                                          (200, 20, 9, 0), (500, 36, 9, 4), (3001, 132, 1009, 4), (700, 260, 40, 2)])
def test_flex16(n, F, V, offset):
    """Mantissas in and out, the largest of them, and what a measuring launch leaves."""
    import torch
    from ngraph_python_b200 import lib
    rng = np.random.RandomState(n)
    idx = rng.randint(0, V, n).astype(np.int16)
    scale, decs = float(np.float32(math.sqrt(F))), (13, 0, 7)
    scales = torch.tensor([[2.0 ** -d, 2.0 ** d] for d in decs], dtype=torch.float32, device="cuda")
    x = torch.from_numpy(idx).cuda()
    raw = lib.raw()

    def device(a):
        t = _off(a.shape, torch.int16, offset)
        t.copy_(torch.from_numpy(a))
        return t

    def check(call, value, shape):
        out = _off(shape, torch.int16, offset)
        stats = torch.zeros((3,), dtype=torch.int32, device="cuda")
        probe = torch.zeros((1,), dtype=torch.int64, device="cuda")
        call(out, stats, probe, 1)
        torch.cuda.synchronize()
        assert not out.any() and not stats.any()
        bits = np.array([int(probe.item()) & 0xffffffff], dtype=np.uint32).view(np.float32)[0]
        assert bits == np.abs(value).max()
        call(out, stats, probe, 0)
        torch.cuda.synchronize()
        want = fx.quantize(value, decs[2])
        assert np.array_equal(out.cpu().numpy(), want)
        assert stats.tolist() == [0, 0, fx.maxabs_stat(want)]

    table = rng.randint(-30000, 30000, (V, F)).astype(np.int16)
    w = device(table)
    step = np.float32(2.0 ** -decs[0])
    check(lambda out, stats, probe, p: lib.check(raw.b2_embed_fprop(
        w.data_ptr(), x.data_ptr(), out.data_ptr(), 1, 3, V, F, n, scale, scales.data_ptr(), 0, 1, 2, stats.data_ptr(), probe.data_ptr(), p, 0)),
        (table[idx].astype(np.float32) * step) * np.float32(scale), (n, F))
    delta = rng.randint(-3000, 3000, (n, F)).astype(np.int16)
    sums = np.zeros((V, F))
    keep = idx != 0
    np.add.at(sums, idx[keep], delta[keep].astype(np.float64))
    assert np.abs(sums).max() < 2 ** 24                      # (exact in fp32)
    d = device(delta)
    nbytes = lib.embed_update_scratch_bytes(V, F, n)
    scratch = torch.full((nbytes,), 0x5A, dtype=torch.uint8, device="cuda")
    check(lambda out, stats, probe, p: lib.check(raw.b2_embed_update(
        d.data_ptr(), x.data_ptr(), out.data_ptr(), 1, 3, V, F, n, scale, 0, 0, scales.data_ptr(), 0, 1, 2, stats.data_ptr(), probe.data_ptr(), p,
        scratch.data_ptr(), nbytes, 0)),
        (sums.astype(np.float32) * step) * np.float32(scale), (V, F))


def _long_sums(n, F):
    """n tokens of which nine in ten are one.  The mantissas of the first half are large and positive, and the second half takes
    them away again but for a few: the sums on the way pass 2^24, beyond which fp32 does not hold every whole number, and
    end where a mantissa holds them."""
    rng = np.random.RandomState(n + F)
    half = n // 2
    idx = np.where(rng.rand(half) < 0.9, 3, rng.randint(0, 11, half))
    first = rng.randint(20000, 32760, (half, F))
    order = rng.permutation(half)
    idx = np.concatenate([idx, idx[order], [5] * (n % 2)]).astype(np.int16)
    delta = np.concatenate([first, rng.randint(-3, 4, (half, F)) - first[order], np.ones((n % 2, F), np.int64)]).astype(np.int16)
    sums = np.zeros((11, F), np.int64)
    np.add.at(sums, idx, delta.astype(np.int64))
    assert np.abs(sums).max() < 32767
    return idx, delta, sums


def test_sums_of_mantissas_that_fp32_does_not_hold():
    """The cases of the next test are such: in parts of 32 that are added in fp32, sums come out wrong."""
    for n, F in ((1600, 64), (4000, 8)):
        idx, delta, sums = _long_sums(n, F)
        rows = delta[idx == 3].astype(np.float32)
        parts = np.array([np.cumsum(rows[k:k + 32], axis=0, dtype=np.float32)[-1] for k in range(0, len(rows), 32)], np.float32)
        way = np.cumsum(parts, axis=0, dtype=np.float32)
        assert np.abs(way).max() > 2 ** 24 - 2 ** 22 and np.any(way[-1] != sums[3])


@pytest.mark.gpu
@pytest.mark.parametrize("n,F,offset", [(256, 8, 0), (257, 8, 0), (1600, 64, 0), (4000, 8, 0), (4000, 36, 0), (4000, 301, 0), (20011, 12, 4), (20011, 12, 1),
                                        (60000, 132, 0)])
def test_flex16_sums_are_exact(n, F, offset):
    import torch
    from ngraph_python_b200 import lib
    idx, delta, sums = _long_sums(n, F)
    scales = torch.ones((3, 2), dtype=torch.float32, device="cuda")
    x, d, out = torch.from_numpy(idx).cuda(), _off((n, F), torch.int16, offset), _off((11, F), torch.int16, offset)
    d.copy_(torch.from_numpy(delta))
    stats, probe = torch.zeros((3,), dtype=torch.int32, device="cuda"), torch.zeros((1,), dtype=torch.int64, device="cuda")
    nbytes = lib.embed_update_scratch_bytes(11, F, n)
    scratch = torch.full((nbytes,), 0x5A, dtype=torch.uint8, device="cuda")
    for measure in (0, 1):
        lib.check(lib.raw().b2_embed_update(d.data_ptr(), x.data_ptr(), out.data_ptr(), 1, 3, 11, F, n, 1.0, -1, 0, scales.data_ptr(), 0, 1, 2,
                                            stats.data_ptr(), probe.data_ptr(), measure, scratch.data_ptr(), nbytes, 0))
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), sums)
    most = np.abs(sums).max()
    assert stats.tolist() == [0, 0, most] and np.array([int(probe.item())], np.uint32).view(np.float32)[0] == most


@pytest.mark.gpu
@pytest.mark.parametrize("dec", [2, 9])
@pytest.mark.parametrize("n", [1, 31, 60, 257, 300])
def test_flex16_index_with_an_exponent(n, dec):
    """Tokens as mantissas of a step below one, of which a single one is no token: what is read beside the list's end is
    none."""
    import torch
    from ngraph_python_b200 import lib
    V, F = 37, 12
    rng = np.random.RandomState(n)
    idx = rng.randint(1, V, n)
    delta = rng.randint(-100, 100, (n, F)).astype(np.int16)
    scales = torch.tensor([[1.0, 1.0], [2.0 ** -dec, 2.0 ** dec], [1.0, 1.0]], dtype=torch.float32, device="cuda")
    x, d = torch.from_numpy((idx << dec).astype(np.int16)).cuda(), torch.from_numpy(delta).cuda()
    out, stats = torch.full((V, F), 7, dtype=torch.int16, device="cuda"), torch.zeros((3,), dtype=torch.int32, device="cuda")
    nbytes = lib.embed_update_scratch_bytes(V, F, n)
    scratch = torch.zeros((nbytes + 4096,), dtype=torch.uint8, device="cuda")
    lib.check(lib.raw().b2_embed_update(d.data_ptr(), x.data_ptr(), out.data_ptr(), 1, 3, V, F, n, 1.0, -1, 0, scales.data_ptr(), 0, 1, 2,
                                        stats.data_ptr(), None, 0, scratch.data_ptr(), nbytes, 0))
    torch.cuda.synchronize()
    want = np.zeros((V, F), np.int64)
    np.add.at(want, idx, delta)
    assert np.array_equal(out.cpu().numpy(), want) and not scratch[nbytes:].any()


@pytest.mark.gpu
def test_recorded_and_replayed_on_another_stream():
    """Two gradients that share a scratch in one graph, replayed with other tokens."""
    import torch
    from ngraph_python_b200 import lib
    V, F, n = 300, 40, 2000
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    idx = torch.randint(0, V, (n,), device="cuda", generator=g)
    deltas = [torch.randint(-8, 9, (n, F), device="cuda", generator=g).float() for _ in range(2)]
    outs = [torch.empty((V, F), device="cuda") for _ in range(2)]
    nbytes = lib.embed_update_scratch_bytes(V, F, n)
    scratch = torch.empty((nbytes,), dtype=torch.uint8, device="cuda")
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()

    def both():
        for d, o in zip(deltas, outs):
            lib.check(lib.raw().b2_embed_update(d.data_ptr(), idx.data_ptr(), o.data_ptr(), 0, 2, V, F, n, 1.0, -1, 0, *PLAIN, scratch.data_ptr(),
                                                nbytes, torch.cuda.current_stream().cuda_stream))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
        with torch.cuda.graph(graph, stream=side):
            both()
        for _ in range(3):
            idx.copy_(torch.randint(0, V, (n,), device="cuda", generator=g))
            graph.replay()
            for d, o in zip(deltas, outs):
                assert torch.equal(o, torch.zeros_like(o).index_add_(0, idx, d))
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls on two streams with a scratch each, beside one another, many times over."""
    import torch
    from ngraph_python_b200 import lib
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    jobs = []
    for V, F, n in ((700, 64, 5000), (3000, 33, 9000)):
        idx = torch.randint(0, V, (n,), device="cuda", generator=g)
        delta = torch.randint(-8, 9, (n, F), device="cuda", generator=g).float()
        nbytes = lib.embed_update_scratch_bytes(V, F, n)
        jobs.append((V, F, n, idx, delta, torch.empty((V, F), device="cuda"), torch.empty((nbytes,), dtype=torch.uint8, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(50):
        for V, F, n, idx, delta, out, scratch, stream in jobs:
            lib.check(lib.raw().b2_embed_update(delta.data_ptr(), idx.data_ptr(), out.data_ptr(), 0, 2, V, F, n, 1.0, -1, 0, *PLAIN, scratch.data_ptr(),
                                                scratch.numel(), stream.cuda_stream))
    torch.cuda.synchronize()
    for V, F, n, idx, delta, out, _, _ in jobs:
        assert torch.equal(out, torch.zeros_like(out).index_add_(0, idx, delta))


@pytest.mark.gpu
def test_large_offsets():
    """A table of more than 2^31 values, its last rows."""
    import torch
    from ngraph_python_b200 import lib
    V, F = 1100001, 2048
    table = torch.empty((V, F), device="cuda")
    table[-3:] = torch.arange(3 * F, device="cuda").view(3, F).float()
    idx = torch.tensor([V - 1, V - 3], dtype=torch.int32, device="cuda")
    out = torch.empty((2, F), device="cuda")
    lib.check(lib.raw().b2_embed_fprop(table.data_ptr(), idx.data_ptr(), out.data_ptr(), 0, 1, V, F, 2, 1.0, *PLAIN, 0))
    assert torch.equal(out, table[idx.long()])
    nbytes = lib.embed_update_scratch_bytes(V, F, 2)
    scratch = torch.empty((nbytes,), dtype=torch.uint8, device="cuda")
    lib.check(lib.raw().b2_embed_update(out.data_ptr(), idx.data_ptr(), table.data_ptr(), 0, 1, V, F, 2, 1.0, -1, 0, *PLAIN, scratch.data_ptr(),
                                        nbytes, 0))
    assert torch.equal(table[idx.long()], out)
    assert int((table != 0).sum()) == int((out != 0).sum())


def test_refusals():
    from ngraph_python_b200 import lib
    raw = lib.raw()
    one = ctypes.c_void_p(256)
    fwd = dict(table=one, idx=one, out=one, flex=0, kind=0, V=4, F=4, n=4)

    def forward(**kw):
        a = dict(fwd, **kw)
        lib.check(raw.b2_embed_fprop(a["table"], a["idx"], a["out"], a["flex"], a["kind"], a["V"], a["F"], a["n"], 1.0, *PLAIN, 0))
    for kw in (dict(V=0), dict(F=-1), dict(n=-1), dict(kind=4), dict(kind=-1), dict(flex=1), dict(kind=3), dict(table=None), dict(idx=None), dict(out=None)):
        with pytest.raises(lib.B200Error, match="error -1"):
            forward(**kw)
    forward(n=0)

    def update(onto=0, nbytes=1 << 20, scratch=one, delta=one, dW=one, flex=0, scales=PLAIN, **kw):
        a = dict(fwd, **kw)
        lib.check(raw.b2_embed_update(delta, a["idx"], dW, flex, a["kind"], a["V"], a["F"], a["n"], 1.0, -1, onto, *scales, scratch, nbytes, 0))
    for kw in (dict(V=0), dict(n=-1), dict(n=1 << 31), dict(kind=9), dict(nbytes=16), dict(scratch=None), dict(delta=None), dict(dW=None), dict(flex=1),
               dict(flex=1, onto=1, scales=(one, 0, 1, 2, one, one, 0)), dict(flex=1, scales=(one, 0, 1, 2, None, one, 0)),
               dict(flex=1, scales=(one, 0, 1, 2, one, None, 1))):
        with pytest.raises(lib.B200Error, match="error -1"):
            update(**kw)


@pytest.mark.parametrize("kind,flex", [(0, 0), (1, 0), (2, 0), (3, 1)])
def test_results_in_the_place_of_operands_are_refused(kind, flex):
    """8 rows of 4 values, 6 tokens; an operand begins or ends a value inside the result, or beside it."""
    from ngraph_python_b200 import lib
    value, token = (2, 2) if flex else (4, {0: 4, 1: 4, 2: 8}[kind])
    form = (256, 0, 1, 2, 256, 256, 0) if flex else PLAIN
    base, table, rows, idx = 1 << 20, 32 * value, 24 * value, 6 * token
    calls = (("overlaps", lambda t, r, x: lib.raw().b2_embed_fprop(t, x, r, flex, kind, 8, 4, 6, 1.0, *form, 0), False),
             ("overlaps", lambda t, r, x: lib.raw().b2_embed_update(r, x, t, flex, kind, 8, 4, 6, 1.0, -1, 0, *form, 256, 1 << 20, 0), True))
    for word, call, of_table in calls:
        def refused(*at):
            with pytest.raises(lib.B200Error) as e:              # (addresses of nothing: refused in any case)
                lib.check(call(*at))
            return word in str(e.value)
        far = base + (1 << 16)
        for r, there in ((base, True), (base + table - value, True), (base + table, False), (base - rows + value, True), (base - rows, False)):
            assert refused(base, r, far) == there
        size, held = (table, lambda x: (base, far, x)) if of_table else (rows, lambda x: (far, base, x))
        for x, there in ((base, True), (base + (size - value) // token * token, True), (base + size, False), (base - idx + token, True), (base - idx, False)):
            assert refused(*held(x)) == there
        # the index is read, and so is the other: they may lie anywhere
        word = "between"
        for at in ((base + 1, far, 2 * far), (base, far + 1, 2 * far), (base, far, 2 * far + 1)):
            assert refused(*at)
        word = "overlaps"


@pytest.mark.gpu
def test_host_memory_is_refused():
    import torch
    from ngraph_python_b200 import lib
    table, idx = torch.zeros((4, 4), device="cuda"), torch.zeros((2,), device="cuda")
    out = torch.zeros((2, 4))
    with pytest.raises(lib.B200Error, match="device memory"):
        lib.check(lib.raw().b2_embed_fprop(table.data_ptr(), idx.data_ptr(), out.data_ptr(), 0, 0, 4, 4, 2, 1.0, *PLAIN, 0))
    there = torch.zeros((2, 4), device="cuda")
    for t, x in ((table.cpu(), idx), (table, idx.cpu())):
        with pytest.raises(lib.B200Error, match="not memory that the device reads"):
            lib.check(lib.raw().b2_embed_fprop(t.data_ptr(), x.data_ptr(), there.data_ptr(), 0, 0, 4, 4, 2, 1.0, *PLAIN, 0))
    nbytes = lib.embed_update_scratch_bytes(4, 4, 2)
    scratch = torch.zeros((nbytes,), dtype=torch.uint8, device="cuda")
    for d, x, s in ((there.cpu(), idx, scratch), (there, idx.cpu(), scratch), (there, idx, scratch.cpu())):
        with pytest.raises(lib.B200Error, match="memory"):
            lib.check(lib.raw().b2_embed_update(d.data_ptr(), x.data_ptr(), table.data_ptr(), 0, 0, 4, 4, 2, 1.0, -1, 0, *PLAIN, s.data_ptr(), nbytes, 0))
    # page-locked memory is read
    pinned = torch.arange(16, dtype=torch.float32).view(4, 4).pin_memory()
    lib.check(lib.raw().b2_embed_fprop(pinned.data_ptr(), idx.data_ptr(), there.data_ptr(), 0, 0, 4, 4, 2, 1.0, *PLAIN, 0))
    torch.cuda.synchronize()
    assert torch.equal(there.cpu(), pinned[:1].expand(2, 4))


@pytest.mark.parametrize("n", [6, 600])
@pytest.mark.parametrize("kind,flex", [(0, 0), (1, 0), (2, 0), (3, 1)])
def test_a_scratch_that_overlaps_is_refused(kind, flex, n):
    from ngraph_python_b200 import lib
    value, token = (2, 2) if flex else (4, {0: 4, 1: 4, 2: 8}[kind])
    form = (64, 0, 1, 2, 64, 64, 0) if flex else PLAIN
    need = lib.embed_update_scratch_bytes(8, 4, n)
    delta, idx, dW = 1 << 20, 2 << 20, 3 << 20
    for at, size in ((delta, n * 4 * value), (idx, n * token), (dW, 32 * value)):
        for scratch, there in ((at, True), (at + size - 1, True), (at + size, False), (at - need + 1, True), (at - need, False)):
            with pytest.raises(lib.B200Error) as e:              # (addresses of nothing: refused in any case)
                lib.check(lib.raw().b2_embed_update(delta, idx, dW, flex, kind, 8, 4, n, 1.0, -1, 0, *form, scratch, need, 0))
            assert ("overlaps" in str(e.value)) == there


def test_exponents_and_statistics_between_addresses_are_refused():
    from ngraph_python_b200 import lib
    raw = lib.raw()
    for flex, kind, form in ((1, 3, (258, 0, 1, 2, 256, 256, 0)), (1, 0, (257, 0, 1, 2, 256, 256, 0)), (0, 3, (258, -1, 1, -1, None, None, 0)),
                             (1, 3, (256, 0, 1, 2, 258, 256, 0)), (1, 3, (256, 0, 1, 2, 256, 260, 1))):
        for call in (lambda: raw.b2_embed_fprop(1 << 20, 2 << 20, 3 << 20, flex, kind, 8, 4, 6, 1.0, *form, 0),
                     lambda: raw.b2_embed_update(1 << 20, 2 << 20, 3 << 20, flex, kind, 8, 4, 6, 1.0, -1, 0, *form, 256, 1 << 20, 0)):
            with pytest.raises(lib.B200Error, match="between two addresses"):
                lib.check(call())


@pytest.mark.gpu
def test_exponents_and_statistics_in_host_memory_are_refused():
    import torch
    from ngraph_python_b200 import lib
    raw = lib.raw()
    table, idx, out = [torch.ones(s, dtype=torch.int16, device="cuda") for s in ((4, 4), (2,), (2, 4))]
    host = np.zeros((64,), np.float32)
    nbytes = lib.embed_update_scratch_bytes(4, 4, 2)
    scratch = torch.zeros((nbytes,), dtype=torch.uint8, device="cuda")
    good = dict(scales=torch.ones((3, 2), device="cuda"), stats=torch.zeros((3,), dtype=torch.int32, device="cuda"),
                probe_out=torch.zeros((1,), dtype=torch.int64, device="cuda"))

    def calls(probe, **moved):
        at = {k: v.data_ptr() for k, v in good.items()}
        at.update(moved)
        form = (at["scales"], 0, 1, 2, at["stats"], at["probe_out"], probe)
        return (lambda: raw.b2_embed_fprop(table.data_ptr(), idx.data_ptr(), out.data_ptr(), 1, 3, 4, 4, 2, 1.0, *form, 0),
                lambda: raw.b2_embed_update(out.data_ptr(), idx.data_ptr(), table.data_ptr(), 1, 3, 4, 4, 2, 1.0, -1, 0, *form, scratch.data_ptr(), nbytes, 0))
    for probe, name in ((0, "scales"), (1, "scales"), (0, "stats"), (1, "probe_out")):
        for call in calls(probe, **{name: host.ctypes.data}):
            with pytest.raises(lib.B200Error, match="memory"):
                lib.check(call())
    # (what is not read or written may be anything)
    for probe, name in ((1, "stats"), (0, "probe_out")):
        for call in calls(probe, **{name: None}):
            lib.check(call())
    torch.cuda.synchronize()
    assert not host.any()
