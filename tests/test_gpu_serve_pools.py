"""Pools without positions: every entry refuses them, none ends the process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import sys
sys.path.insert(0, {root!r})
import torch
import tcb_b200 as T
from tcb_b200 import serve
ctx = T.Context(0)
i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
q = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
x, s = torch.zeros(2, 128, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
pool = torch.zeros(4, 2, 16, 64, dtype=torch.float16, device="cuda")
for k in (torch.empty(4, 2, 0, 64, dtype=torch.float16, device="cuda"), pool[:, :, :0], pool[:, :, :12]):
    p = serve.Pages(ctx, k, k)
    for call in (lambda: p.append(x, x, s), lambda: p.attend(q, q, i([0, 1, 2]), i([1, 1]), i([[0], [0]]), 1, 16),
                 lambda: p.attend_prefix(q, q, i([0]), 1, i([1, 1]), i([[0], [0]]), 16)):
        try:
            call()
        except T.TcbError as e:
            assert e.code in (1, 3), e.code
        else:
            raise AssertionError("taken")
print("done")
"""


def test_pools_without_positions():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", SCRIPT.format(root=root)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), (r.returncode, r.stderr[-2000:])
