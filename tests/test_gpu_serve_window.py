"""Pages that no row sees need not be there: a server gives the pages between
the first positions and the window back, in every form of the attention."""
import math

import pytest
import torch

import tcb_b200 as T
from tcb_b200 import serve

from test_gpu_serve import BF16, F16, attn_case, check_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    torch.cuda.set_device(0)
    return T.Context(0)


def seen_pages(n, rows, page, window, sinks):
    """pages that hold a position some row of the request sees"""
    out = set()
    for p in range(n - rows, n):
        w = max(0, p - window + 1)
        out |= {j // page for j in range(w, p + 1)} | {j // page for j in range(min(sinks, p + 1))}
    return out


@pytest.mark.parametrize("most", [700, 1 << 20])  # row by row where the rows are few, by tiles
@pytest.mark.parametrize("rows", [1, 3, 90, 300])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(50, 0), (50, 4), (1, 17), (130, 40), (0, 5), (0, 200), (0, 0)])
def test_pages_out_of_sight_are_not_looked_up(ctx, most, rows, page, window, sinks):
    lens, m = [700, 333, 611], [rows, min(rows, 200), 1]
    dtype = F16 if rows % 2 else BF16
    c = attn_case(lens, m, 8, 2, 64 if page == 32 else 128, page, dtype, seed=page + rows)
    t = c["tables"].clone()
    for b, (n, r) in enumerate(zip(lens, m)):
        seen = seen_pages(n, r, page, window, sinks)
        for j in range(-(-n // page)):
            if j not in seen:
                t[b, j] = (-1, 2 ** 31 - 1)[j % 2]
    out = torch.full_like(c["q"], math.nan)
    ctx.device_error(clear=True)
    serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], out, c["row_start"], c["kv_len"], t, rows if most == 700 else 400, most, window=window, sinks=sinks)
    assert ctx.device_error(clear=True) == 0
    check_rows(out, c, lens, m, dtype, window, sinks, 1 / math.sqrt(c["q"].shape[2]), "given back")
