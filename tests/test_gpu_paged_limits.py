"""Paged operators at the limits of a launch and of its waits, on a B200."""
import importlib
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_paged import BF16, DEV, F16, ints

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


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_tile_idle_for_seconds(dtype):
    """One tile of a CTA without rows in an item that takes the other longer (3 s and more) than a wait for a unit may,
    and with rows in the next item.  148 heads for 148 CTAs: the last one works on the end of the long request's last
    item, then on all items of the short one.  The long request's keys are one block, repeated."""
    paged = importlib.import_module("index-tts-25-metal_b200.paged")
    heads, dim, bs, keys = 148, 128, 128, 3 * 2 ** 27
    k = torch.zeros(1, bs, heads, dim, dtype=dtype, device=DEV)
    q = torch.ones(128 + 300, heads, dim, dtype=dtype, device=DEV)
    table = torch.zeros(2, keys // bs, dtype=torch.int32, device=DEV)
    out = paged.attention(q, k, k, table, ints([keys, 300]), ints([0, 128, 428]), 300)
    assert (out == 0).all()
