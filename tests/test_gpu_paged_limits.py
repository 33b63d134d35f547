"""Paged operators at the limits of a launch, on a B200."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FIRST = """
import importlib, sys
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
from test_gpu_paged import TableState, run_tables
paged = importlib.import_module("index-tts-25-metal_b200.paged")
for n in {counts}:
    s = TableState([(11 * i) % 70 for i in range(n)], [(i % 3) - 1 for i in range(n)], 16, spare=1)
    d = s.device()
    run_tables(paged, d, 16)
    s.check(d)
"""


@pytest.mark.parametrize("counts", [[3045, 3046], [3071], [3073], [8192, 3060]])
def test_tables_of_many_requests_are_the_first_call_of_a_process(counts):
    """A request takes 16 bytes of the kernel's shared memory, so that these counts lie about the 48 KB beyond which a
    launch needs leave: no call may rely on an earlier, larger one to have got it."""
    run = subprocess.run([sys.executable, "-c", FIRST.format(root=ROOT, counts=counts)], capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
