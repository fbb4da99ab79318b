"""Which places of tensors of heads are taken and which are refused, and what the arguments of a call may not do to the process."""
import subprocess
import sys

import pytest

from ngraph_python_b200 import lib

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
    done = subprocess.run([sys.executable, "-c", NO_ROWS % positions], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
    assert "overlap" not in done.stdout and "one place" not in done.stdout, done.stdout
