"""Rows of q outside every request cost no scratch."""
import math

import pytest
import torch

import tcb_b200 as T
from tcb_b200 import serve

from test_gpu_serve import BF16, F16, attn_case, check_rows

pytestmark = pytest.mark.gpu


def test_attend_few_rows_of_a_large_batch():
    """200 rows of 8 million, their positions in parts: partial results for the
    rows that are there."""
    ctx, n, rows, T_ = T.Context(0), 3000, 200, 1 << 23
    c = attn_case([n], [rows], 1, 1, 64, 64, BF16, seed=21)
    q = torch.zeros(T_, 1, 64, dtype=BF16, device="cuda")
    q[:rows] = c["q"]
    out = torch.full_like(q, 3.0)
    serve.Pages(ctx, c["k"], c["v"]).attend(q, out, c["row_start"], c["kv_len"], c["tables"], rows, 1 << 20)
    assert ctx.device_error(clear=True) == 0
    check_rows(out[:rows], c, [n], [rows], BF16, None, 0, 1 / 8, "padded")
    assert (out[rows:] == 3).all()


@pytest.mark.parametrize("pad", [0, 5, 4000])
@pytest.mark.parametrize("H,KVH,hd", [(1, 1, 64), (6, 2, 128)])
def test_attend_requests_in_a_padded_batch(pad, H, KVH, hd):
    """Requests that start anywhere in the rows, parts of the positions joined."""
    ctx, lens, m = T.Context(0), [900, 1, 1500, 333], [61, 1, 0, 90]
    c = attn_case(lens, m, H, KVH, hd, 32, F16, seed=H)
    n = sum(m)
    q = torch.zeros(n + 2 * pad, H, hd, dtype=F16, device="cuda")
    q[pad:pad + n] = c["q"]
    out = torch.full_like(q, 3.0)
    serve.Pages(ctx, c["k"], c["v"]).attend(q, out, c["row_start"] + pad, c["kv_len"], c["tables"], 95, 1 << 20)
    assert ctx.device_error(clear=True) == 0
    check_rows(out[pad:pad + n], c, lens, m, F16, None, 0, 1 / math.sqrt(hd), "padded")
    assert (out[:pad] == 3).all() and (out[pad + n:] == 3).all()
