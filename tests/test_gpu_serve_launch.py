"""Launches of the logits' penalties that need more shared memory than a kernel
has without asking, aligned and unaligned in either order, each order in a
process of its own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
SCRIPT = """
import sys
sys.path[:0] = [{here!r}, {root!r}]
import torch
import tcb_b200 as T
from test_gpu_serve import logits_case, run_logits, check_logits
ctx = T.Context(0)
for xt in (torch.float32, torch.float16, torch.bfloat16):
    for ot in (torch.float32, torch.float16, torch.bfloat16):
        for V in {sizes}:
            c = logits_case(160, V, 9, seed=V, n_bias=5, n_masks=2, dtype=xt)
            check_logits(c, *run_logits(ctx, c, out_dtype=ot))
assert ctx.device_error() == 0
print("done")
"""


@pytest.mark.parametrize("sizes", [(1000, 1001), (1001, 1000)])
def test_penalize_large_tiles_in_either_order(sizes):
    """160 rows: tiles of 512 threads, 64 KB with biases; rows of 1000 logits are
    read four at a time, rows of 1001 one by one."""
    text = SCRIPT.format(here=HERE, root=os.path.dirname(HERE), sizes=sizes)
    r = subprocess.run([sys.executable, "-c", text], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stderr[-2000:]
