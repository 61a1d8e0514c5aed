"""fence_paged_plan at the request counts where its shared memory passes what a kernel may use without asking, and its report
of contexts out of range."""
import os
import subprocess
import sys

import pytest

from test_kv8_gpu import T, run_plan  # noqa: F401  (T is a fixture)

pytestmark = pytest.mark.gpu

# In a process of its own for each: a larger call before would have asked for the memory already.
CHILD = """
import os, sys
sys.path.insert(0, sys.argv[1])
import conftest, kv8_ref, test_kv8_gpu as t
import torch
fb, n = conftest.load_pkg(), int(sys.argv[2])
t.check_plan(fb, torch, kv8_ref, [i % 40 for i in range(n)], [(1, 0, 17, -1, 1)[i % 5] for i in range(n)], 16, 5, 500)
"""


@pytest.mark.parametrize("n", [2036, 2037, 2047, 2048])
def test_first_plan_of_a_process(n):
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", CHILD, here, str(n)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("ctx", [-1, -2 ** 31, 4 * 16 + 1, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [-1, 0, 1])
def test_contexts_out_of_range_are_reported(fb, T, ctx, new):  # noqa: F811
    """A negative context, or one longer than its row of the table; the requests beside it are served. One of full length is in
    range."""
    table, free = [[0, 1, 2, 3], [4, -3, -3, -3], [-3, -3, -3, -3]], [5, 6, 7, 8, 9]
    got = run_plan(fb, T, [ctx, 16, 0], [new, 1, 2], table, free, 8, 16, 4, 10)
    assert fb.lib().fence_device_error() == -1
    assert got["kv_len"][1:] == [17, 2]
    got = run_plan(fb, T, [64, 16, 0], [0, 1, 2], table, free, 8, 16, 4, 10)
    assert fb.lib().fence_device_error() == 0 and got["kv_len"] == [64, 17, 2]
