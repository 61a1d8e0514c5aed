"""fence_paged_plan at the request counts where its shared memory passes what a kernel may use without asking."""
import os
import subprocess
import sys

import pytest

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
