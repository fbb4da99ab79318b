"""Which places of tensors of heads are taken and which are refused, and what the arguments of a call may not do to the process."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from ngraph_python_b200 import lib
from oracle import heads_oracle as ho

NO_ROWS = """
import ctypes
from ngraph_python_b200 import lib
a = lib.HeadsArgs(rows=0, head_dim=8, rotary_dim=8, parts=1, turns=1 << 20, positions=%s, position_kind=2, position_count=1, position_group=1, amplitude=1.0)
a.part[0].heads, a.part[0].weight = 2, 1 << 21
g = lib.HeadsGrads()
g.part[0].d_weight = 1 << 22
n = lib.heads_bprop_scratch_bytes(a)
print(lib.raw().b2_heads_bprop(ctypes.byref(a), ctypes.byref(g), 1 << 30, n, None), lib.raw().b2_last_error().decode())
"""


@pytest.mark.parametrize("positions", ["(1 << 30) + 256", "1 << 30", "(1 << 22) + 8"])
def test_no_rows_and_positions_in_a_results_memory(positions):
    """Positions of no rows are no memory: nothing to overlap, and nothing to divide by.  (A process of its own, which a signal would end.)"""
    done = subprocess.run([sys.executable, "-c", NO_ROWS % positions], capture_output=True, text=True, timeout=300,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
    assert "overlap" not in done.stdout and "one place" not in done.stdout, done.stdout


def _places(base, R, heads, D, row, head):
    """The addresses of a tensor's values, in values."""
    return set(base + r * row + h * head + i for r in range(R) for h in range(heads) for i in range(D))


def _answer(R, D, tensors):
    """What b2_heads_fprop says of these (x, out) tensors, (base, heads, row, head) each, in values; bases from 2^28 on."""
    a = lib.HeadsArgs(rows=R, head_dim=D, rotary_dim=0, parts=len(tensors), amplitude=1.0)
    for p, ((x, heads, x_row, x_head), (out, _, out_row, out_head)) in zip(a.part, tensors):
        p.heads, p.x, p.x_row, p.x_head, p.out, p.out_row, p.out_head = heads, 4 * x, x_row, x_head, 4 * out, out_row, out_head
    return lib.raw().b2_heads_fprop(ctypes.byref(a), None), lib.raw().b2_last_error().decode()


def _overlap(rc, text):
    return rc == -1 and ("overlap" in text or "in one place" in text or "place of an operand" in text)


AT = 1 << 28


@pytest.mark.parametrize("layout", ["heads next to one another", "in wider rows", "heads first"])
def test_queries_and_keys_between_one_anothers_heads(layout):
    """[rows][heads][queries, keys, values]: each result in its operand's place, or both in another tensor of that layout."""
    R, H, D = 4, 3, 8
    row, head = {"heads next to one another": (3 * H * D, 3 * D), "in wider rows": (3 * H * D + 40, 3 * D), "heads first": (3 * D, 3 * R * D)}[layout]
    for far in (0, 1 << 20):
        tensors = [((AT + i * D, H, row, head), (AT + far + i * D, H, row, head)) for i in range(2)]
        assert not _overlap(*_answer(R, D, tensors)), _answer(R, D, tensors)
        # one head of keys, between those of the queries; and one value into them
        one = [tensors[0], ((AT + D, 1, row, head), (AT + far + D, 1, row, head))]
        assert not _overlap(*_answer(R, D, one))
        for off in (-1, 1 - D):
            one[1] = ((AT + D + off, 1, row, head), (AT + far + D + off, 1, row, head))
            assert _overlap(*_answer(R, D, one))


def test_overlaps_are_found_as_one_by_one():
    """Two results of the same strides, wherever they begin: refused where a value has two owners, and only there."""
    rng = np.random.RandomState(0)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        R, D, heads = rng.randint(1, 5), rng.randint(1, 6), [rng.randint(1, 4), rng.randint(1, 4)]
        most = max(heads)
        if rng.randint(2):
            head = D * rng.randint(1, 4) + rng.randint(0, 2)
            row = most * head + rng.randint(0, 5) * D
        else:
            row = D * rng.randint(1, 4) + rng.randint(0, 2)
            head = R * row + rng.randint(0, 5) * D
        bases = [AT, AT + rng.randint(-2 * row - 2 * head, 2 * row + 2 * head + 1)]
        tensors = [((AT + (1 << 20) * (1 + i), h, row, head), (b, h, row, head)) for i, (h, b) in enumerate(zip(heads, bases))]
        both = [_places(b, R, h, D, row, head) for h, b in zip(heads, bases)]
        assert all(len(p) == R * h * D for p, h in zip(both, heads))
        meets = bool(both[0] & both[1])
        rc, text = _answer(R, D, tensors)
        assert _overlap(rc, text) == meets, (R, D, heads, row, head, bases, text)
        seen[meets] += 1
    assert min(seen.values()) > 500


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["in wider rows", "heads first"])
@pytest.mark.parametrize("D", [16, 18])
def test_rotations_between_one_anothers_heads(layout, D):
    """Queries and keys of [rows][heads][queries, keys, values] rotated where they lie; the values stay.  A rotation is off by at
    most six halves of a step of |u| + |v| (see the tests of the rotation)."""
    import torch
    R, H = 37, 3
    row, head = {"in wider rows": (3 * H * D + 40, 3 * D), "heads first": (3 * D, 3 * R * D)}[layout]
    size = (R - 1) * row + (H - 1) * head + 3 * D
    whole = np.random.RandomState(0).standard_normal(size).astype(np.float32)
    on = torch.from_numpy(whole).cuda()
    turns = lib.rotary_turns(D)
    turns_on = turns.cuda()
    a = lib.HeadsArgs(rows=R, head_dim=D, rotary_dim=D, parts=2, turns=turns_on.data_ptr(), amplitude=1.0, position_count=R, position_group=1)
    for i in range(2):
        p = a.part[i]
        p.heads, p.x, p.out = H, on.data_ptr() + 4 * i * D, on.data_ptr() + 4 * i * D
        p.x_row, p.x_head, p.out_row, p.out_head = row, head, row, head
    lib.check(lib.raw().b2_rotary(ctypes.byref(a), 0, None, None, None, 0, None))
    got = on.cpu().numpy()
    angle = ho.angles(np.arange(R), turns.numpy())
    at = np.arange(R)[:, None, None] * row + np.arange(H)[:, None] * head + np.arange(D)
    rest = np.ones(size, bool)
    for i in range(2):
        want, terms = ho.rotate(whole[at + i * D], angle, D, False)
        assert np.all(np.abs(got[at + i * D] - want) <= 6 * 2.0 ** -24 * terms)
        rest[at + i * D] = False
    assert np.array_equal(got[rest], whole[rest])
