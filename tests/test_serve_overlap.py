"""tcb_page_plan refuses arrays that overlap: its grid reads the inputs while
the outputs are written.  The addresses of the refused calls are never followed."""
import pytest
import torch

import tcb_b200 as T
from tcb_b200 import serve

import serve_ref as R
from test_serve import UNSUPPORTED, ctx, plan  # noqa: F401 (ctx is a fixture)

OUT = ("row_start", "kv_len", "slots", "positions", "balance", "taken")
AT = dict(cached=0x100, fresh=0x200, tables=0x300, free=0x400, n_free=0x500, row_start=0x600, kv_len=0x700, slots=0x800, positions=0x900, balance=0xA00)


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("other", ["cached", "fresh", "free", "n_free", "tables"])
def test_an_output_in_an_input(ctx, out, other):  # noqa: F811
    assert plan(ctx, **{out: AT[other]}) == UNSUPPORTED


@pytest.mark.parametrize("a", OUT)
@pytest.mark.parametrize("b", OUT[:5])
def test_two_outputs_in_one_place(ctx, a, b):  # noqa: F811
    if a != b:
        assert plan(ctx, **{a: AT[b]}) == UNSUPPORTED


@pytest.mark.parametrize("kw", [
    dict(kv_len=0x104), dict(kv_len=0xF8 + 4), dict(balance=0x41C), dict(taken=0x700 + 4), dict(row_start=0x700 - 8), dict(row_start=0x4FC),
    dict(free=0x310), dict(n_free=0x31C), dict(slots=0x708 - 16), dict(ldt=64, balance=0x400 + 12), dict(ldt=64, cached=0x400 - 4, free=0x1400),
    dict(ldt=64, free_cap=80, free=0x300 + 16)])
def test_in_part(ctx, kw):  # noqa: F811
    assert plan(ctx, **kw) == UNSUPPORTED


@pytest.mark.gpu
def test_side_by_side_is_taken():
    """Arrays that end where others begin, and outputs between the rows of the tables."""
    ctx, B, rows = T.Context(0), 3, 20
    buf = torch.full((200,), -7, dtype=torch.int32, device="cuda")
    wide = buf[:60].view(3, 20)
    tables = wide[:, :4]  # 16 entries between the rows
    row_start, taken = buf[4:8], buf[8:9]  # the first row's
    cached, fresh, kv_len, free, n_free, balance, positions = (buf[a:b] for a, b in ((60, 63), (63, 66), (66, 69), (69, 79), (79, 80), (80, 81), (81, 101)))
    slots = buf[102:142].view(torch.int64)
    tables.fill_(-1)
    tables[1, 0] = 40
    for t, v in ((cached, [0, 15, 16]), (fresh, [5, 2, 9]), (free, list(range(10))), (n_free, [10])):
        t.copy_(torch.tensor(v, dtype=torch.int32))
    tables[2, 0] = 41
    before = tables.tolist()
    serve.plan(ctx, 16, cached, fresh, tables, free, n_free, row_start, kv_len, slots, positions, balance, taken)
    want = R.plan(16, [0, 15, 16], [5, 2, 9], before, list(range(10)), 10, rows)
    got = [t.tolist() for t in (tables, row_start, kv_len, slots, positions)] + [balance.item(), taken.item()]
    assert got == list(want)
    assert (wide[1:, 4:] == -7).all() and (wide[0, 9:] == -7).all() and (buf[142:] == -7).all() and buf[101] == -7
    for kw in (dict(kv_len=cached), dict(kv_len=fresh), dict(balance=n_free), dict(positions=buf[60:80]), dict(slots=buf[0:40].view(torch.int64))):
        a = dict(kv_len=kv_len, slots=slots, positions=positions, balance=balance)
        a.update(kw)
        with pytest.raises(T.TcbError) as e:
            serve.plan(ctx, 16, cached, fresh, tables, free, n_free, row_start, a["kv_len"], a["slots"], a["positions"], a["balance"], taken)
        assert e.value.code == UNSUPPORTED
    assert ctx.device_error() == 0
