"""The operators of a language model's training step and of its serving calls that this backend has
beside the reference's: what a pass of each computes, over the sizes such programs use.

  embed       a table lookup with a scale: out[t] = scale * table[token[t]], and its gradient, the rows
              of delta added up per token in the order of the tokens -- as a whole table of sums, or
              onto a gradient that another use of the table (the output layer) has already left there
  norm        the edge between two blocks: the block's result is normalised, gated and added to the
              scaled residual stream, which is normalised again for the next block,
                  stream = a * residual + gate * rms(block) * w_post,   out = rms(stream) * w_pre
              and the gradients of all of it from those of `out` and `stream`
  adamw       one AdamW step over every tensor of a model, with its two moments in 32 bits, or in 8
              (e4m3 values with one scale per 256, the second one as its square root, rounded at
              random from a hash of the position and the step)

Tensors are fp32; the table lookups take flex16 (int16 mantissas, one exponent per tensor) as well.
"""
import ctypes
import math

import numpy as np
import torch

own = False


def _lib():
    from ngraph_python_b200 import lib
    return lib


def listed():
    return [
        # serving: the tokens of a small batch, one each
        dict(name="embed_16x512", kind="embed", grad=False, flex=False, tokens=16, features=512, vocab=32000, idx="f32"),
        # a training batch
        dict(name="embed_16384x1024", kind="embed", grad=False, flex=False, tokens=16384, features=1024, vocab=32000, idx="i64"),
        # its gradient as a table of its own: rows of tokens that do not occur are zero
        dict(name="embed_grad_8192x1024", kind="embed", grad=True, flex=False, tokens=8192, features=1024, vocab=32000, idx="f32", onto=False),
        # ... and added to the gradient of an output layer that shares the table
        dict(name="embed_grad_onto_16384x768", kind="embed", grad=True, flex=False, tokens=16384, features=768, vocab=50000, idx="i64", onto=True),
        # int16 mantissas, odd sizes
        dict(name="embed_grad_flex16_3001x301", kind="embed", grad=True, flex=True, tokens=3001, features=301, vocab=10007, idx="f32", onto=False),
        # serving, one sequence: the edge between two blocks for one token
        dict(name="norm_1x2048", kind="norm", grad=False, rows=1, features=2048, block=True, post=True, gate="feature"),
        # a training batch between two blocks
        dict(name="norm_8192x4096", kind="norm", grad=False, rows=8192, features=4096, block=True, post=True, gate="feature"),
        # gradients: odd sizes with a gate for every row (a router's weight), and the training batch
        dict(name="norm_grad_777x1001", kind="norm", grad=True, rows=777, features=1001, block=True, post=True, gate="row"),
        dict(name="norm_grad_8192x4096", kind="norm", grad=True, rows=8192, features=4096, block=True, post=True, gate="feature"),
        # the update of a small model, where the launch counts, and of one with eighty million values
        dict(name="adamw32_small", kind="adamw", bits=32, layers=2, features=64, vocab=1000),
        dict(name="adamw32_large", kind="adamw", bits=32, layers=12, features=640, vocab=32000),
        dict(name="adamw8_large", kind="adamw", bits=8, layers=12, features=640, vocab=32000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "norm", "adamw"])
    if kind == "embed":
        features = _log(rng, 64, 2048)
        if rng.random() < 0.6:
            features = max(64, features // 8 * 8)
        vocab = _log(rng, 200, min(50000, (1 << 25) // features))
        grad = rng.random() < 0.6
        flex = rng.random() < 0.3
        return dict(kind=kind, grad=grad, flex=flex, tokens=_log(rng, 1, min(16384, (1 << 24) // features)), features=features,
                    vocab=vocab, idx="f32" if flex else rng.choice(["f32", "i32", "i64"]),
                    onto=bool(grad and not flex and rng.random() < 0.4))
    if kind == "norm":
        features = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            features = max(64, features // 16 * 16)
        block = rng.random() < 0.8
        return dict(kind=kind, grad=rng.random() < 0.5, rows=_log(rng, 1, min(16384, (1 << 25) // features)), features=features,
                    block=block, post=bool(block and rng.random() < 0.6),
                    gate=rng.choice(["none", "feature", "row", "full"]) if block else "none")
    features = _log(rng, 16, 640)
    return dict(kind=kind, bits=rng.choice([8, 32]), layers=rng.randint(1, 12), features=features, vocab=_log(rng, 100, 32000))


# ---- the work -----------------------------------------------------------------------------------------
def _sizes(case):
    """(values, decayed) of every tensor of the model: a table, and per layer four matrices and four vectors."""
    f = case["features"]
    found = [(case["vocab"] * f, True)]
    for _ in range(case["layers"]):
        found += [(f, False), (3 * f * f, True), (f * f, True), (f, False), (4 * f * f, True), (4 * f, False), (4 * f * f, True), (f, False)]
    return found


def _spread(case):
    """The chance of each token: as k ** -1 over the table, like words of a text."""
    edges = np.log(np.arange(1, case["vocab"] + 2))
    return np.diff(edges) / edges[-1]


def _distinct(case):
    return float(np.sum(-np.expm1(case["tokens"] * np.log1p(-np.minimum(_spread(case), 1 - 1e-9)))))


def work(case):
    if case["kind"] == "embed":
        size = 2 if case["flex"] else 4
        n, f = case["tokens"], case["features"]
        index = n * {"f32": size, "i32": 4, "i64": 8}[case["idx"]]
        if not case["grad"]:
            return {"bytes": index + (n + _distinct(case)) * f * size, "flops": n * f}
        table = 2 * _distinct(case) if case["onto"] else case["vocab"]
        return {"bytes": index + (n + table) * f * size, "flops": 2 * n * f}
    if case["kind"] == "norm":
        t, f = case["rows"], case["features"]
        gate = {"none": 0, "feature": f, "row": t, "full": t * f}[case["gate"]]
        vectors = f * (1 + case["post"])
        if not case["grad"]:
            tensors = 4 if case["block"] else 2
            return {"bytes": 4 * (tensors * t * f + gate + vectors + t * (1 + case["post"])), "flops": (14 if case["block"] else 4) * t * f}
        tensors = 6 if case["block"] else 4
        return {"bytes": 4 * (tensors * t * f + 2 * gate + 2 * vectors + t * (1 + case["post"])), "flops": (30 if case["block"] else 12) * t * f}
    n = sum(s for s, _ in _sizes(case))
    if case["bits"] == 32:
        return {"bytes": 28 * n, "flops": 15 * n}
    return {"bytes": 16 * n + 16 * (n / 256), "flops": 40 * n}


# ---- what a program has in hand --------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


_IDX = {"f32": (torch.float32, 0), "i32": (torch.int32, 1), "i64": (torch.int64, 2), "i16": (torch.int16, 3)}


def _prepare_embed(case, seed):
    g = _generator(seed)
    n, f, v, flex = case["tokens"], case["features"], case["vocab"], case["flex"]
    u = torch.rand((n,), device="cuda", generator=g, dtype=torch.float64)
    tokens = (torch.pow(float(v + 1), u) - 1).floor().clamp_(0, v - 1).long()
    state = dict(case=case, scale=math.sqrt(f), pad=0 if case["grad"] else -1)
    kind = "i16" if flex else case["idx"]
    state["idx"] = tokens.to(_IDX[kind][0]) if not flex else tokens.clamp_(max=32767).to(torch.int16)
    if flex:
        # rows of the exponent table (step, 1 / step): the operand, the index, the result
        dec = (14, 0, 8)
        state["steps"] = torch.tensor([[2.0 ** -d, 2.0 ** d] for d in dec], device="cuda")
        state["stats"] = torch.zeros((3,), dtype=torch.int32, device="cuda")
    make = (lambda *s: _randn(g, *s).mul_(3000).round_().clamp_(-32767, 32767).to(torch.int16)) if flex else (lambda *s: _randn(g, *s))
    kinds = torch.int16 if flex else torch.float32
    if case["grad"]:
        state["delta"] = make(n, f)
        state["out"] = _randn(g, v, f) if case["onto"] else torch.empty((v, f), dtype=kinds, device="cuda")
    else:
        state["table"] = make(v, f)
        state["out"] = torch.empty((n, f), dtype=kinds, device="cuda")
    if own:
        lib = _lib()
        scales = (state["steps"].data_ptr(), 0, 1, 2, state["stats"].data_ptr(), None, 0) if flex else (None, -1, -1, -1, None, None, 0)
        if case["grad"]:
            nbytes = lib.embed_update_scratch_bytes(v, f, n)
            state["scratch"] = torch.empty((nbytes,), dtype=torch.uint8, device="cuda")
            state["call"] = lib.raw().b2_embed_update
            state["args"] = (state["delta"].data_ptr(), state["idx"].data_ptr(), state["out"].data_ptr(), int(flex), _IDX[kind][1], v, f, n,
                             state["scale"], state["pad"], int(case["onto"])) + scales + (state["scratch"].data_ptr(), nbytes)
        else:
            state["call"] = lib.raw().b2_embed_fprop
            state["args"] = (state["table"].data_ptr(), state["idx"].data_ptr(), state["out"].data_ptr(), int(flex), _IDX[kind][1], v, f, n,
                             state["scale"]) + scales
    return state


def _prepare_norm(case, seed):
    g = _generator(seed)
    t, f = case["rows"], case["features"]
    s = dict(case=case, eps=1e-6, a=0.9 if case["block"] else 1.0)
    s["residual"] = _randn(g, t, f).mul_(2.0)
    s["pre"] = 1.0 + 0.1 * _randn(g, f)
    if case["block"]:
        s["block"] = _randn(g, t, f)
        s["post"] = 1.0 + 0.1 * _randn(g, f) if case["post"] else None
        shape = {"none": None, "feature": (1, f), "row": (t, 1), "full": (t, f)}[case["gate"]]
        s["gate"] = None if shape is None else 0.5 + 0.2 * _randn(g, *shape)
    else:
        s["block"] = s["post"] = s["gate"] = None
    if case["grad"]:
        s["d_out"], s["d_stream"] = _randn(g, t, f), _randn(g, t, f)
        # what the forward pass has left
        x = s["residual"].double()
        if case["block"]:
            u = s["block"].double()
            if case["post"]:
                rho = (u.square().mean(1, keepdim=True) + s["eps"]).rsqrt()
                s["block_rstd"] = rho.float()
                u = u * rho * s["post"]
            x = s["a"] * x + (u if s["gate"] is None else u * s["gate"])
        s["stream"] = x.float()
        s["stream_rstd"] = (x.square().mean(1, keepdim=True) + s["eps"]).rsqrt().float()
        del x
        s["grads"] = {k: torch.empty_like(s[k]) for k in ("residual", "block", "gate", "post", "pre") if s.get(k) is not None}
    else:
        s["stream"] = torch.empty_like(s["residual"]) if case["block"] else None
        s["out"] = torch.empty_like(s["residual"])
        s["stream_rstd"] = torch.empty((t, 1), device="cuda")
        if case["post"]:
            s["block_rstd"] = torch.empty((t, 1), device="cuda")
    if own:
        lib = _lib()
        at = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        a = lib.NormArgs()
        a.rows, a.features, a.gate_kind = t, f, {"none": 0, "feature": 1, "row": 2, "full": 3}[case["gate"]]
        a.residual_scale, a.eps = s["a"], s["eps"]
        a.block_stride = a.residual_stride = a.stream_stride = a.gate_stride = a.out_stride = f
        a.block, a.gate, a.post_weight, a.pre_weight = at(s["block"]), at(s["gate"]), at(s["post"]), at(s["pre"])
        a.residual, a.stream, a.out = at(s["residual"]), at(s["stream"]), at(s.get("out"))
        a.block_rstd, a.stream_rstd = at(s.get("block_rstd")), at(s["stream_rstd"])
        s["norm"] = a
        if case["grad"]:
            if not case["block"]:
                a.stream = None
            d = lib.NormGrads()
            d.d_out, d.d_stream = at(s["d_out"]), at(s["d_stream"])
            d.d_out_stride = d.d_stream_stride = d.d_residual_stride = d.d_block_stride = d.d_gate_stride = f
            d.d_residual, d.d_block, d.d_gate = [at(s["grads"].get(k)) for k in ("residual", "block", "gate")]
            d.d_post_weight, d.d_pre_weight = at(s["grads"].get("post")), at(s["grads"]["pre"])
            s["norm_grads"] = d
            s["scratch_bytes"] = lib.norm_bprop_scratch_bytes(a)
            s["scratch"] = torch.empty((s["scratch_bytes"],), dtype=torch.uint8, device="cuda")
    return s


BLOCK = 256         # values with one scale
TOP = 448.0         # the largest e4m3 value
LEAST = 2.0 ** -9   # the smallest
TINY = 2.0 ** -100  # blocks whose largest value is not above this are held as zeros


def _prepare_adamw(case, seed):
    g = _generator(seed)
    # the tensors lie in one arena, each from a multiple of 256 values on, as an exchange of gradients lays them out
    starts, total = [], 0
    for size, _ in _sizes(case):
        starts.append(total)
        total += -(-size // BLOCK) * BLOCK
    live = torch.zeros((total,), dtype=torch.bool, device="cuda")
    decay = torch.zeros((total,), device="cuda")
    for (size, decayed), at in zip(_sizes(case), starts):
        live[at:at + size] = True
        decay[at:at + size] = float(decayed)
    make = lambda s: _randn(g, total).mul_(s).mul_(live)  # noqa: E731
    s = dict(case=case, decay=decay, param=make(0.05), grad=make(1e-3), t=1000, seed=seed & 0x7fffffff,
             lr=3e-4, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.1)
    m, r = make(3e-4), make(1e-3).abs_()
    if case["bits"] == 32:
        s["m"], s["v"] = m, r.square_()
    else:
        for name, x in (("m", m), ("r", r)):
            top = x.view(-1, BLOCK).abs().amax(1)
            s[name + "_scale"] = top / TOP
            s[name] = torch.where(top[:, None] > 0, x.view(-1, BLOCK) * (TOP / top[:, None]), 0.0).clamp_(-TOP, TOP).to(torch.float8_e4m3fn).view(-1)
    if own:
        lib = _lib()
        tensors = (lib.AdamwTensor * len(starts))()
        for x, (size, decayed), at in zip(tensors, _sizes(case), starts):
            x.param, x.grad = s["param"].data_ptr() + 4 * at, s["grad"].data_ptr() + 4 * at
            x.n, x.decay, x.counter = size, float(decayed), at & 0xffffffff
            if case["bits"] == 32:
                x.m, x.v = s["m"].data_ptr() + 4 * at, s["v"].data_ptr() + 4 * at
            else:
                x.m, x.v = s["m"].data_ptr() + at, s["r"].data_ptr() + at
                x.m_scales, x.v_scales = [s[k].data_ptr() + 4 * (at // BLOCK) for k in ("m_scale", "r_scale")]
        nbytes, chunks = lib.adamw_plan_bytes(tensors, case["bits"])
        s["plan"] = torch.empty((nbytes,), dtype=torch.uint8, device="cuda")
        lib.adamw_plan(tensors, case["bits"], s["plan"].data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
        s["step"] = torch.full((1,), float(s["t"]), device="cuda")
        s["hyper"] = lib.AdamwHyper(s["lr"], s["beta1"], s["beta2"], s["eps"], s["wd"])
        s["args"] = (s["plan"].data_ptr(), chunks, case["bits"], ctypes.byref(s["hyper"]), None, None, s["step"].data_ptr(), s["seed"])
    return s


def prepare(case, seed):
    return {"embed": _prepare_embed, "norm": _prepare_norm, "adamw": _prepare_adamw}[case["kind"]](case, seed)


# ---- one pass --------------------------------------------------------------------------------------------
def _stored(s, value):
    """Results as flex16 holds them: mantissas, rounded to the nearest even one, and the largest of them."""
    m = torch.round(value * s["steps"][2, 1]).clamp(-32768, 32767)
    s["stats"][2] = torch.maximum(s["stats"][2], m.abs().amax().int())
    s["out"].copy_(m.to(torch.int16))
    return [s["out"], s["stats"]]


def _plain_embed(s):
    case, flex = s["case"], s["case"]["flex"]
    tokens = s["idx"].long()
    if not case["grad"]:
        rows = s["table"][tokens]
        if flex:
            return _stored(s, rows.float() * s["steps"][0, 0] * s["scale"])
        s["out"].copy_(rows * s["scale"])
        return [s["out"]]
    keep = (tokens != s["pad"])[:, None]
    if flex:
        # (sums of mantissas are whole numbers: exact)
        sums = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda").index_add_(0, tokens, s["delta"].double() * keep)
        return _stored(s, sums.float() * s["steps"][0, 0] * s["scale"])
    sums = torch.zeros_like(s["out"]).index_add_(0, tokens, s["delta"] * keep)
    if case["onto"]:
        s["out"].add_(sums * s["scale"])
    else:
        s["out"].copy_(sums * s["scale"])
    return [s["out"]]


def _rstd(x, eps):
    return 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)


def _plain_norm(s):
    x = s["residual"]
    if s["block"] is not None:
        u = s["block"]
        if s["post"] is not None:
            s["block_rstd"].copy_(_rstd(u, s["eps"]))
            u = u * s["block_rstd"] * s["post"]
        if s["gate"] is not None:
            u = u * s["gate"]
        x = s["stream"].copy_(s["a"] * x + u)
    s["stream_rstd"].copy_(_rstd(x, s["eps"]))
    s["out"].copy_(x * s["stream_rstd"] * s["pre"])
    return [v for v in (s["out"], s["stream"], s["stream_rstd"], s.get("block_rstd")) if v is not None]


def _through_rms(d, x, rstd, w):
    """The gradients of x and w where y = x * rstd * w and d is the gradient of y."""
    xhat = x * rstd
    dx = d * w
    return rstd * (dx - xhat * (dx * xhat).mean(1, keepdim=True)), (d * xhat).sum(0)


def _plain_norm_grad(s):
    found = s["grads"]
    dx, dw = _through_rms(s["d_out"], s["stream"], s["stream_rstd"], s["pre"])
    found["pre"].copy_(dw)
    dx = dx + s["d_stream"]
    found["residual"].copy_(s["a"] * dx)
    if s["block"] is not None:
        u = s["block"] if s["post"] is None else s["block"] * s["block_rstd"] * s["post"]
        du = dx
        if s["gate"] is not None:
            dg = dx * u
            shared = {"feature": 0, "row": 1}.get(s["case"]["gate"])
            found["gate"].copy_(dg if shared is None else dg.sum(shared, keepdim=True))
            du = dx * s["gate"]
        if s["post"] is not None:
            du, dw = _through_rms(du, s["block"], s["block_rstd"], s["post"])
            found["post"].copy_(dw)
        found["block"].copy_(du)
    return dict(found)


def _mix(x):
    """Thirty-two bits from thirty-two, in wrapping int32."""
    shifted = lambda v, k: (v >> k) & ((1 << (32 - k)) - 1)  # noqa: E731
    x = (x ^ shifted(x, 16)) * (0x9E3779B9 - (1 << 32))
    x = (x ^ shifted(x, 15)) * (0xBB67AE85 - (1 << 32))
    return x ^ shifted(x, 16)


def _to_e4m3(q, bits):
    """|q| <= 448 to one of its two neighbours among the e4m3 values, the upper one with the chance that 16 random bits give it."""
    a = q.abs().clamp(max=TOP)
    low = a < 2.0 ** -6
    b = torch.where(low, a + 2.0 ** -6, a)
    c = ((b.view(torch.int32) + (bits << 4)) & ~0xFFFFF).view(torch.float32)
    return torch.where(low, c - 2.0 ** -6, c)


def _plain_adamw(s):
    s["t"] += 1
    f32 = lambda x: float(np.float32(x))  # noqa: E731
    b1, b2, c1, c2 = f32(s["beta1"]), f32(s["beta2"]), f32(1 - s["beta1"]), f32(1 - s["beta2"])
    size = f32(s["lr"] / (1 - s["beta1"] ** s["t"]))
    root = f32(1 / math.sqrt(1 - s["beta2"] ** s["t"]))
    keep = 1.0 - s["decay"] * f32(s["lr"] * s["wd"])
    g, eight = s["grad"], s["case"]["bits"] == 8
    if eight:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        r = (s["r"].float().view(-1, BLOCK) * s["r_scale"][:, None]).view(-1)
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * c1
    v = v * b2 + (g * g) * c2
    r = torch.sqrt(v)
    s["param"].copy_(s["param"] * keep - (m / (r * root + f32(s["eps"]))) * size)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return dict(param=s["param"], m=s["m"], v=s["v"])
    key = _mix(torch.full((1,), (s["seed"] + 0x9E3779B9 * s["t"] + (1 << 31)) % (1 << 32) - (1 << 31), dtype=torch.int32, device="cuda"))
    h = _mix(torch.arange(m.numel(), dtype=torch.int32, device="cuda") ^ key)
    for name, x, bits in (("m", m, h & 0xFFFF), ("r", r, (h >> 16) & 0xFFFF)):
        top = x.view(-1, BLOCK).abs().amax(1)
        inverse = torch.where(top > TINY, TOP / top, 0.0)
        q = (x.view(-1, BLOCK) * inverse[:, None]).view(-1)
        c = _to_e4m3(q, bits)
        if name == "r":
            c = torch.where((q > 0) & (c < LEAST), LEAST, c)
        s[name].copy_(torch.copysign(c, q).to(torch.float8_e4m3fn))
        s[name + "_scale"].copy_(torch.where(top > TINY, top / TOP, 0.0))
    return dict(param=s["param"], m=s["m"], m_scale=s["m_scale"], r=s["r"], r_scale=s["r_scale"])


def run(state):
    kind = state["case"]["kind"]
    if not own:
        if kind == "embed":
            return _plain_embed(state)
        if kind == "adamw":
            return _plain_adamw(state)
        return _plain_norm_grad(state) if state["case"]["grad"] else _plain_norm(state)
    lib, stream = _lib(), torch.cuda.current_stream().cuda_stream
    if kind == "embed":
        lib.check(state["call"](*state["args"], stream))
        return [state["out"], state["stats"]] if state["case"]["flex"] else [state["out"]]
    if kind == "adamw":
        lib.check(lib.raw().b2_adamw_step(*state["args"], stream))
        names = ("param", "m", "v") if state["case"]["bits"] == 32 else ("param", "m", "m_scale", "r", "r_scale")
        return {k: state[k] for k in names}
    if state["case"]["grad"]:
        lib.check(lib.raw().b2_norm_bprop(ctypes.byref(state["norm"]), ctypes.byref(state["norm_grads"]), state["scratch"].data_ptr(),
                                          state["scratch_bytes"], stream))
        return dict(state["grads"])
    lib.check(lib.raw().b2_norm_fprop(ctypes.byref(state["norm"]), stream))
    return [v for v in (state["out"], state["stream"], state["stream_rstd"], state.get("block_rstd")) if v is not None]


# ---- the same in 64 bits, from the definitions ---------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = lambda k: None if s.get(k) is None else s[k].double()  # noqa: E731
    if case["kind"] == "embed":
        if case["flex"]:
            return None             # whole numbers
        tokens = s["idx"].long()
        if not case["grad"]:
            return [d("table").index_select(0, tokens) * s["scale"]]
        # sums per token over the sorted tokens
        order = torch.argsort(tokens, stable=True)
        rows = d("delta").index_select(0, order)
        found, counts = torch.unique_consecutive(tokens[order], return_counts=True)
        ends = counts.cumsum(0)
        run_up = torch.cat([torch.zeros((1, case["features"]), dtype=torch.float64, device="cuda"), rows.cumsum(0)])
        sums = run_up[ends] - run_up[ends - counts]
        sums[found == s["pad"]] = 0.0
        table = d("out") if case["onto"] else torch.zeros((case["vocab"], case["features"]), dtype=torch.float64, device="cuda")
        table[found] += sums * s["scale"]
        return [table]
    if case["kind"] == "norm":
        eps = s["eps"]
        u, w, x = d("block"), d("post"), d("residual")
        if not case["grad"]:
            rho = None
            if u is not None:
                if w is not None:
                    rho = torch.rsqrt(torch.einsum("tf,tf->t", u, u) / case["features"] + eps)[:, None]
                    u = torch.einsum("tf,tx,f->tf", u, rho, w)
                x = s["a"] * x + (u if s["gate"] is None else u * d("gate"))
            rstd = torch.rsqrt(torch.einsum("tf,tf->t", x, x) / case["features"] + eps)[:, None]
            out = torch.einsum("tf,tx,f->tf", x, rstd, d("pre"))
            return [v for v in (out, x if u is not None else None, rstd, rho) if v is not None]
        # by the automatic derivatives of the forward formula, at the stored stream
        found = {}
        x = d("stream").requires_grad_()
        pre = d("pre").requires_grad_()
        out = x * d("stream_rstd").detach() * pre
        # (the stored reciprocal deviation is an input: its own derivative, -rstd^3 x / F, is added by hand)
        gx, found["pre"] = torch.autograd.grad(out, (x, pre), d("d_out"))
        rstd = d("stream_rstd")
        with torch.no_grad():
            x = x.detach()
            dot = torch.einsum("tf,tf,f->t", d("d_out"), x, d("pre"))[:, None]
            gx = gx - rstd.pow(3) * x * dot / case["features"] + d("d_stream")
            found["residual"] = s["a"] * gx
            if u is not None:
                gate = d("gate")
                rho = d("block_rstd") if w is not None else None
                value = u if w is None else u * rho * w
                if gate is not None:
                    found["gate"] = {"feature": lambda: torch.einsum("tf,tf->f", gx, value)[None], "row": lambda: torch.einsum("tf,tf->t", gx, value)[:, None],
                                     "full": lambda: gx * value}[case["gate"]]()
                    gx = gx * gate
                if w is not None:
                    found["post"] = torch.einsum("tf,tf,tx->f", gx, u, rho)
                    dot = torch.einsum("tf,tf,f->t", gx, u, w)[:, None]
                    gx = gx * rho * w - rho.pow(3) * u * dot / case["features"]
                found["block"] = gx
        return found
    t = s["t"] + 1
    g = d("grad")
    if case["bits"] == 32:
        m, v = d("m"), d("v")
    else:
        m = (d("m").view(-1, BLOCK) * d("m_scale")[:, None]).view(-1)
        v = (d("r").view(-1, BLOCK) * d("r_scale")[:, None]).view(-1).square()
    m = s["beta1"] * m + (1 - s["beta1"]) * g
    v = s["beta2"] * v + (1 - s["beta2"]) * g * g
    step = s["lr"] * (m / (1 - s["beta1"] ** t)) / (torch.sqrt(v / (1 - s["beta2"] ** t)) + s["eps"])
    param = d("param") * (1 - s["lr"] * s["wd"] * d("decay")) - step
    if case["bits"] == 32:
        return dict(param=param, m=m, v=v)
    # (values rounded at random have no such value)
    return dict(param=param, m=None, m_scale=None, r=None, r_scale=None)
