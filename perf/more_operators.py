"""Operators that a transformer's training step and its serving calls need around their matrix products, and
the optimizer of those products' weights, over the sizes that such programs use.

  rotary      queries and keys rotated by their position: feature pairs (halves of the head, or neighbours) of
              the first `rotary` features of a head turn by position * frequency, the others pass through; the
              frequencies may be stretched for contexts longer than those of the training; the gradient is the
              rotation back
  heads       a norm of every head of the queries and keys with the rotation in the same pass,
                  out = rotated(x / sqrt(mean(x^2) + eps) * w),
              w shared by the heads of a tensor, and its gradients
  muon        one step of an optimizer that orthogonalises the update of every matrix: with m the running mean of
              the gradients, u = (1 - mu) g + mu m and x = u / |u|, five times
                  a = x x^T,   x = 3.4445 x + (-4.7750 a + 2.0315 a a) x
              and param = param (1 - lr decay) - lr scale x

Tensors are fp32.
"""
import ctypes
import math

import torch

own = False

EPS = 1e-6
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _lib():
    from ngraph_python_b200 import lib
    return lib


def _heads(name, kind, rows, q, k, dim, rotary, **more):
    """q and k: how many heads the queries and the keys have; sequence: positions run from `first` on over so many rows."""
    case = dict(name=name, kind=kind, grad=False, rows=rows, q=q, k=k, dim=dim, rotary=rotary, pairs="halves", positions="i64", first=0,
                sequence=rows, scaling="none", fused=False)
    case.update(more)
    return case


def listed():
    return [
        # serving: one new token of each of sixteen sequences, far into their contexts
        _heads("rotary_16x32x128", "rotary", 16, 32, 8, 128, 128, sequence=1, first=30000),
        # a training batch, four sequences, stretched for longer contexts; queries and keys lie in one product's rows
        _heads("rotary_8192x16x128", "rotary", 8192, 16, 4, 128, 128, sequence=2048, scaling="parts", fused=True),
        # the gradient at odd sizes, neighbours paired, a part of the head rotated, positions of the framework's own type
        _heads("rotary_grad_3001x12x80", "rotary", 3001, 12, 12, 80, 40, grad=True, pairs="neighbours", positions="f32"),
        # a long prompt at positions beyond a million, stretched evenly
        _heads("rotary_32768x8x64", "rotary", 32768, 8, 2, 64, 64, pairs="neighbours", first=1 << 20, scaling="linear"),
        # serving: one new token of each of sixteen sequences
        _heads("heads_16x32x128", "heads", 16, 32, 8, 128, 128, sequence=1, first=5000, fused=True),
        # a training batch, four sequences
        _heads("heads_8192x32x128", "heads", 8192, 32, 8, 128, 128, sequence=2048, fused=True),
        # gradients: odd sizes with a part of the head rotated, and the training batch
        _heads("heads_grad_777x12x96", "heads", 777, 12, 4, 96, 48, grad=True, pairs="neighbours", positions="i32"),
        _heads("heads_grad_8192x32x128", "heads", 8192, 32, 8, 128, 128, grad=True, sequence=2048),
        # the matrices of a small model, where launches count
        dict(name="muon_small", kind="muon", shapes="2*64x192 2*64x64 2*64x256 2*256x64"),
        # odd and thin matrices next to one another
        dict(name="muon_ragged", kind="muon", shapes="3*301x1001 1001x301 2*77x77 1x640 129x1 1000x777"),
        # models of forty-nine million values and of a hundred million in wide layers
        dict(name="muon_12x640", kind="muon", shapes="12*640x1920 12*640x640 12*640x2560 12*2560x640"),
        dict(name="muon_2x2048", kind="muon", shapes="2*2048x6144 2*2048x2048 2*2048x8192 2*8192x2048"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "heads", "muon"])
    if kind == "muon":
        parts, left = [], 6.0e7         # values of all matrices
        for _ in range(rng.randint(1, 5)):
            r, c = _log(rng, 1, 2048), _log(rng, 1, 2048)
            if rng.random() < 0.5:
                r, c = max(16, r // 16 * 16), max(16, c // 16 * 16)
            count = rng.randint(1, max(1, min(12, int(left / (r * c)))))
            left -= count * r * c
            parts.append("%d*%dx%d" % (count, r, c))
        return dict(kind=kind, shapes=" ".join(parts))
    dim = _log(rng, 16, 256)
    if rng.random() < 0.6:
        dim = max(16, dim // 16 * 16)
    rotary = dim // 2 * 2 if rng.random() < 0.6 else max(2, dim // 4 * 2)
    k = _log(rng, 1, 8)
    q = k * rng.choice([1, 2, 3, 4])
    rows = _log(rng, 1, min(32768, (1 << 25) // ((q + k) * dim)))
    return dict(kind=kind, grad=rng.random() < 0.5, rows=rows, q=q, k=k, dim=dim, rotary=rotary, pairs=rng.choice(["halves", "neighbours"]),
                positions=rng.choice(["i64", "i32", "f32"]), first=rng.choice([0, _log(rng, 1, 1 << 20)]), sequence=rng.choice([1, rows, _log(rng, 1, rows)]),
                scaling=rng.choice(["none", "linear", "base", "parts"]), fused=rng.random() < 0.5)


# ---- the work -----------------------------------------------------------------------------------------
def _shapes(case):
    """(count, rows, columns) of every stack of matrices."""
    found = []
    for text in case["shapes"].split():
        count, _, shape = text.rpartition("*")
        r, c = shape.split("x")
        found.append((int(count or 1), int(r), int(c)))
    return found


_POSITIONS = {"f32": (torch.float32, 0, 4), "i32": (torch.int32, 1, 4), "i64": (torch.int64, 2, 8)}


def work(case):
    if case["kind"] == "muon":
        nbytes = flops = 0
        for count, r, c in _shapes(case):
            n, m = min(r, c), max(r, c)
            nbytes += 20 * count * r * c
            flops += 5 * count * (3 * n * n * m + n ** 3)       # (both squares are symmetric: half of each)
        return {"bytes": nbytes, "flops": flops}
    heads, dim = case["q"] + case["k"], case["dim"]
    values = case["rows"] * heads * dim
    more = _POSITIONS[case["positions"]][2] * case["rows"] + 4 * case["rotary"]
    if case["kind"] == "rotary":
        return {"bytes": 8 * values + more, "flops": 3 * values * case["rotary"] / dim}
    if not case["grad"]:
        return {"bytes": 8 * values + more + 4 * case["rows"] * heads + 8 * dim, "flops": 8 * values}
    return {"bytes": 12 * values + more + 4 * case["rows"] * heads + 16 * dim, "flops": 18 * values}


# ---- what a program has in hand --------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


BASE, FACTOR, ORIGINAL, LOW, HIGH = 10000.0, 8.0, 2048.0, 1.0, 32.0


def _frequencies(case):
    """Radians a position of every pair, in 64 bits, and what the rotated features are multiplied by."""
    d = case["rotary"]
    i = torch.arange(d // 2, dtype=torch.float64)
    base = BASE
    if case["scaling"] == "base" and d > 2:
        base = BASE * FACTOR ** (d / (d - 2))
    f = base ** (-2 * i / d)
    if case["scaling"] == "linear":
        f = f / FACTOR
    if case["scaling"] == "parts":
        # pairs that turn often over the original context keep their frequency, those that do not are stretched
        keep = ((ORIGINAL * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / FACTOR
    return f.cuda(), 0.1 * math.log(FACTOR) + 1.0 if case["scaling"] == "parts" else 1.0


def _prepare_heads(case, seed):
    g = _generator(seed)
    rows, dim = case["rows"], case["dim"]
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    s = dict(case=case)
    s["frequencies"], s["amplitude"] = _frequencies(case)
    # each sequence goes on from its own place
    sequence = case["sequence"]
    starts = torch.randint(0, 64, (-(-rows // sequence),), device="cuda", generator=g) + case["first"]
    at = torch.arange(rows, device="cuda")
    s["positions"] = (starts[at // sequence] + at % sequence).to(_POSITIONS[case["positions"]][0])
    given = "d_out" if case["grad"] else "x"
    tensors = {given}
    if case["kind"] == "heads":
        tensors |= {"x"}
    for name in sorted(tensors):
        if case["fused"]:       # the rows of one product: queries, keys and values of all heads
            whole = randn(rows, case["q"] + 2 * case["k"], dim)
            s[name] = [whole[:, :case["q"]], whole[:, case["q"]:case["q"] + case["k"]]]
        else:
            s[name] = [randn(rows, case["q"], dim), randn(rows, case["k"], dim)]
    s["out"] = [torch.empty((rows, h, dim), device="cuda") for h in (case["q"], case["k"])]
    if case["kind"] == "heads":
        s["weight"] = [1.0 + 0.1 * randn(dim) for _ in "qk"]
        s["rstd"] = [torch.empty((rows, h), device="cuda") for h in (case["q"], case["k"])]
        if case["grad"]:        # (what the forward pass has left)
            for x, r in zip(s["x"], s["rstd"]):
                r.copy_((x.double().square().mean(2) + EPS).rsqrt())
            s["d_weight"] = [torch.empty((dim,), device="cuda") for _ in "qk"]
    if own:
        lib = _lib()
        s["turns"] = lib.rotary_turns(case["rotary"], BASE, case["scaling"], FACTOR, ORIGINAL, LOW, HIGH).cuda()
        a = lib.HeadsArgs()
        a.rows, a.head_dim, a.rotary_dim = rows, dim, case["rotary"]
        a.interleaved, a.inverse = int(case["pairs"] == "neighbours"), int(case["grad"] and case["kind"] == "rotary")
        a.turns, a.amplitude, a.eps, a.parts = s["turns"].data_ptr(), s["amplitude"], EPS, 2
        a.positions, a.position_kind = s["positions"].data_ptr(), _POSITIONS[case["positions"]][1]
        a.position_count, a.position_group = rows, 1
        backward = case["kind"] == "heads" and case["grad"]
        for i in range(2):
            p, x = a.part[i], s["x" if backward else given][i]
            p.heads, p.x, p.x_row, p.x_head = x.shape[1], x.data_ptr(), x.stride(0), x.stride(1)
            if not backward:
                p.out, p.out_row, p.out_head = s["out"][i].data_ptr(), s["out"][i].stride(0), dim
            if case["kind"] == "heads":
                p.weight, p.rstd = s["weight"][i].data_ptr(), s["rstd"][i].data_ptr()
        s["args"] = a
        if backward:
            d = lib.HeadsGrads()
            for i in range(2):
                p, x = d.part[i], s["d_out"][i]
                p.d_out, p.d_out_row, p.d_out_head = x.data_ptr(), x.stride(0), x.stride(1)
                p.d_x, p.d_x_row, p.d_x_head = s["out"][i].data_ptr(), s["out"][i].stride(0), dim
                p.d_weight = s["d_weight"][i].data_ptr()
            s["grads"] = d
            s["scratch_bytes"] = lib.heads_bprop_scratch_bytes(a)
            s["scratch"] = torch.empty((s["scratch_bytes"],), dtype=torch.uint8, device="cuda")
    return s


def _prepare_muon(case, seed):
    g = _generator(seed)
    s = dict(case=case, lr=0.02, mu=0.95, eps=1e-7, wd=0.01, param=[], grad=[], mean=[], scale=[])
    for count, r, c in _shapes(case):
        make = lambda k: torch.randn((count, r, c), device="cuda", generator=g).mul_(k)  # noqa: E731
        # gradients of a few directions that weigh more than the others, as those of a batch do
        some = min(r, c, 8)
        strong = torch.randn((count, r, some), device="cuda", generator=g) @ torch.randn((count, some, c), device="cuda", generator=g)
        s["param"].append(make(1.0 / math.sqrt(r)))
        s["grad"].append(make(1e-3) + strong.mul_(1e-3))
        s["mean"].append(make(3e-4) + strong * 0.3)
        s["scale"].append(math.sqrt(max(1.0, r / c)))
    if own:
        lib = _lib()
        matrices = (lib.MuonMatrix * sum(x.shape[0] for x in s["param"]))()
        k = 0
        for i, (count, r, c) in enumerate(_shapes(case)):
            for j in range(count):
                x = matrices[k]
                k += 1
                x.param, x.grad, x.mean = [s[key][i][j].data_ptr() for key in ("param", "grad", "mean")]
                x.rows, x.cols, x.decay, x.scale = r, c, 1.0, s["scale"][i]
        s["sizes"] = lib.muon_plan_sizes(matrices)
        s["plan"] = torch.empty((s["sizes"].plan_bytes,), dtype=torch.uint8, device="cuda")
        s["scratch"] = torch.empty((s["sizes"].scratch_bytes,), dtype=torch.uint8, device="cuda")
        lib.muon_plan(matrices, s["plan"].data_ptr(), s["sizes"].plan_bytes, torch.cuda.current_stream().cuda_stream)
        s["hyper"] = lib.MuonHyper(s["lr"], s["mu"], s["eps"], s["wd"], *COEFFICIENTS, 5, 1)
        s["args"] = (s["plan"].data_ptr(), ctypes.byref(s["sizes"]), ctypes.byref(s["hyper"]), None, None, None, s["scratch"].data_ptr(),
                     s["sizes"].scratch_bytes, None)
    return s


def prepare(case, seed):
    return _prepare_muon(case, seed) if case["kind"] == "muon" else _prepare_heads(case, seed)


# ---- one pass --------------------------------------------------------------------------------------------
def _turned(s, x, cos, sin):
    """x [rows, heads, dim] with its pairs turned."""
    d = s["case"]["rotary"]
    first, second = (slice(0, d // 2), slice(d // 2, d)) if s["case"]["pairs"] == "halves" else (slice(0, d, 2), slice(1, d, 2))
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., second] * cos + x[..., first] * sin
    out[..., d:] = x[..., d:]
    return out


def _angles(s):
    angle = s["positions"].double()[:, None, None] * s["frequencies"]       # [rows, 1, pairs]
    return (torch.cos(angle) * s["amplitude"]).float(), (torch.sin(angle) * s["amplitude"]).float()


def _plain_heads(s):
    case, found = s["case"], {}
    cos, sin = _angles(s)
    if case["kind"] == "rotary":
        x = s["d_out" if case["grad"] else "x"]
        if case["grad"]:
            sin = -sin
        return {"q": s["out"][0].copy_(_turned(s, x[0], cos, sin)), "k": s["out"][1].copy_(_turned(s, x[1], cos, sin))}
    for i, name in ((0, "q"), (1, "k")):
        x, w, rstd, out = s["x"][i], s["weight"][i], s["rstd"][i], s["out"][i]
        if not case["grad"]:
            rstd.copy_(1.0 / torch.sqrt((x * x).mean(2) + EPS))
            found[name] = out.copy_(_turned(s, x * rstd[..., None] * w, cos, sin))
            found[name + "_rstd"] = rstd
            continue
        d = _turned(s, s["d_out"][i], cos, -sin)
        xhat = x * rstd[..., None]
        found[name + "_weight"] = s["d_weight"][i].copy_((d * xhat).sum((0, 1)))
        d = d * w
        found[name] = out.copy_(rstd[..., None] * (d - xhat * (d * xhat).mean(2, keepdim=True)))
    return found


def _orthogonal(x):
    """Five steps for a stack of matrices that have no more rows than columns."""
    a, b, c = COEFFICIENTS
    for _ in range(5):
        square = x @ x.mT
        x = a * x + (b * square + c * (square @ square)) @ x
    return x


def _plain_muon(s):
    for param, grad, mean, scale in zip(s["param"], s["grad"], s["mean"], s["scale"]):
        mean.copy_(s["mu"] * mean + (1 - s["mu"]) * grad)
        u = (1 - s["mu"]) * grad + s["mu"] * mean
        u = u / (u.double().square().sum((1, 2), keepdim=True).sqrt().float() + s["eps"])
        u = _orthogonal(u.mT).mT if u.shape[1] > u.shape[2] else _orthogonal(u)
        param.copy_(param * (1 - s["lr"] * s["wd"]) - (s["lr"] * scale) * u)
    return dict(param=s["param"], mean=s["mean"])


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return _plain_muon(state) if kind == "muon" else _plain_heads(state)
    lib, stream = _lib(), torch.cuda.current_stream().cuda_stream
    if kind == "muon":
        lib.check(lib.raw().b2_muon_step(*state["args"], stream))
        return dict(param=state["param"], mean=state["mean"])
    a, q, k = ctypes.byref(state["args"]), state["out"][0], state["out"][1]
    if kind == "rotary":
        lib.check(lib.raw().b2_rotary(a, 0, None, None, None, 0, stream))
        return dict(q=q, k=k)
    if state["case"]["grad"]:
        lib.check(lib.raw().b2_heads_bprop(a, ctypes.byref(state["grads"]), state["scratch"].data_ptr(), state["scratch_bytes"], stream))
        return dict(q=q, k=k, q_weight=state["d_weight"][0], k_weight=state["d_weight"][1])
    lib.check(lib.raw().b2_heads_fprop(a, stream))
    return dict(q=q, k=k, q_rstd=state["rstd"][0], k_rstd=state["rstd"][1])


# ---- the same in 64 bits, from the definitions ---------------------------------------------------------------
def _exact_turned(case, x, turn):
    """Pairs as complex numbers, multiplied by turn [rows, 1, pairs]."""
    d = case["rotary"]
    head, rest = x[..., :d], x[..., d:]
    if case["pairs"] == "halves":
        z = torch.complex(*head.chunk(2, -1)) * turn
        return torch.cat([z.real, z.imag, rest], -1)
    z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), rest], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "muon":
        found = dict(param=[], mean=[])
        a, b, c = COEFFICIENTS
        for param, grad, mean, scale in zip(s["param"], s["grad"], s["mean"], s["scale"]):
            mean = torch.lerp(grad.double(), mean.double(), s["mu"])
            u = torch.lerp(grad.double(), mean, s["mu"])
            u = u / (torch.linalg.matrix_norm(u, keepdim=True) + s["eps"])
            tall = u.shape[1] > u.shape[2]
            # every step multiplies x by a polynomial of x x^T, which commutes with those of the other steps: their product first
            square = u.mT @ u if tall else u @ u.mT
            eye = torch.eye(square.shape[-1], dtype=torch.float64, device="cuda")
            product = eye
            for _ in range(5):
                step = a * eye + b * square + c * (square @ square)
                product = step @ product
                square = step @ square @ step
            x = u @ product if tall else product @ u
            found["param"].append(param.double() - s["lr"] * (s["wd"] * param.double() + scale * x))
            found["mean"].append(mean)
        return found
    angle = torch.einsum("r,p->rp", s["positions"].double(), s["frequencies"])[:, None]
    turn = torch.polar(torch.full_like(angle, s["amplitude"]), angle)
    found = {}
    for i, name in ((0, "q"), (1, "k")):
        if case["kind"] == "rotary":
            found[name] = _exact_turned(case, s["d_out" if case["grad"] else "x"][i].double(), turn.conj() if case["grad"] else turn)
            continue
        x, w = s["x"][i].double().requires_grad_(case["grad"]), s["weight"][i].double().requires_grad_(case["grad"])
        rstd = torch.rsqrt(torch.linalg.vector_norm(x, dim=2).square() / case["dim"] + EPS)
        out = _exact_turned(case, torch.einsum("rhd,rh,d->rhd", x, rstd, w), turn)
        if case["grad"]:
            found[name], found[name + "_weight"] = torch.autograd.grad(out, (x, w), s["d_out"][i].double())
        else:
            found[name], found[name + "_rstd"] = out, rstd
    return found
