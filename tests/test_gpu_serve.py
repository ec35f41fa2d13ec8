"""The serving operators on the GPU against plain 64-bit restatements
(tests/serve_ref.py): the page plan, the append, attention over the pages
(windows, first positions, ragged rows, single rows, a shared prefix) and the
logits' penalties and pick."""
import math
import random

import pytest
import torch

import tcb_b200 as T
from tcb_b200 import serve

import serve_ref as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
BOUNDS = 9


@pytest.fixture(scope="module")
def ctx():
    torch.cuda.set_device(0)
    return T.Context(0)


@pytest.fixture(autouse=True)
def no_device_error(ctx):
    ctx.device_error(clear=True)
    yield
    assert ctx.device_error(clear=True) == 0


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------ page plan

def run_plan(ctx, page, cached, fresh, tables, free, n_free, rows):
    B = len(cached)
    t = i32(tables).view(B, -1)
    rs, kl, balance, taken = i32([-9] * (B + 1)), i32([-9] * B), i32([-9]), i32([-9])
    sl, ps = torch.full((rows,), -9, dtype=torch.int64, device="cuda"), i32([-9] * rows)
    for _ in range(2):  # the same call again gives the same
        serve.plan(ctx, page, i32(cached), i32(fresh), t, i32(free), i32([n_free]), rs, kl, sl, ps, balance, taken)
    return t.tolist(), rs.tolist(), kl.tolist(), sl.tolist(), ps.tolist(), balance.item(), taken.item()


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("B,max_fresh,tight", [(1, 1, False), (1, 0, False), (7, 1, False), (33, 90, False), (64, 1, True), (257, 40, True),
                                               (1000, 3, False), (8192, 2, True)])
def test_plan(ctx, page, B, max_fresh, tight):
    r = random.Random(B * page + max_fresh)
    cached = [r.choice([0, r.randint(0, 5 * page), page, page - 1, page + 1]) for _ in range(B)]
    fresh = [r.randint(0, max_fresh) for _ in range(B)]
    if B > 6:
        cached[3], fresh[4] = -1, -2  # refused
        cached[5] = 8 * page  # too long for its table with any new position
    have = [-(-max(c, 0) // page) for c in cached]
    need = sum(-(-(c + f) // page) - -(-c // page) for c, f in zip(cached, fresh) if c >= 0 and f > 0)
    ids = list(range(sum(have) + need + 5))
    r.shuffle(ids)
    tables = [[ids.pop() if j < h else -1 for j in range(8)] for h in have]
    n_free = need // 2 if tight else len(ids) - 1
    rows = sum(max(f, 0) for f in fresh) + (3 if B % 2 else -1 if B > 6 and fresh[-1] > 0 else 0)
    rows = max(rows, 0)
    want = R.plan(page, cached, fresh, tables, ids, n_free, rows)
    got = run_plan(ctx, page, cached, fresh, tables, ids, n_free, rows)
    for name, g, w in zip(("tables", "row_start", "kv_len", "slots", "positions", "balance", "taken"), got, want):
        assert g == w, name


def test_plan_free_count_is_held_to_the_list(ctx):
    want = R.plan(16, [0, 0], [16, 16], [[-1], [-1]], [5], 1, 32)
    assert run_plan(ctx, 16, [0, 0], [16, 16], [[-1], [-1]], [5], 99, 32)[1:] == want[1:]
    assert run_plan(ctx, 16, [0], [1], [[-1]], [5], -3, 1)[2:] == ([0], [-1], [-1], 0, 0)


def test_plan_of_nothing(ctx):
    e, left = i32([]), i32([7])
    serve.plan(ctx, 16, e, e, e.view(0, 0), i32([1, 2]), i32([2]), i32([3]), e, torch.full((4,), 5, dtype=torch.int64, device="cuda")[:0], e, left)
    assert left.item() == 2


def test_tensors_that_are_not_what_is_wanted(ctx):
    """Refused before anything is launched: types, sizes, strides, places."""
    k, v = pools(4, 2, 16, 64, F16, fill=0.0)
    p = serve.Pages(ctx, k, v)
    q, rs, kl, t = torch.zeros(2, 4, 64, device="cuda", dtype=F16), i32([0, 1, 2]), i32([3, 4]), i32([[0], [1]])
    x, s = torch.zeros(2, 128, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    lg, f = torch.zeros(2, 40, device="cuda"), torch.zeros(2, device="cuda")
    i = i32([0, 0, 0])
    refused = [lambda: p.attend(q, q, rs.long(), kl, t, 1, 16), lambda: p.attend(q, q, rs[:2], kl, t, 1, 16), lambda: p.attend(q, q, rs, kl.cpu(), t, 1, 16),
               lambda: p.attend(q, q[:1], rs, kl, t, 1, 16), lambda: p.attend(q[..., :32], q[..., :32], rs, kl, t, 1, 16), lambda: p.attend(q, q, rs, kl, t[:1], 1, 16),
               lambda: p.attend(q.transpose(0, 1), q.transpose(0, 1), rs, kl, t, 1, 16), lambda: p.attend(q, q, rs, kl, t, 1, 16, window=-2), lambda: p.attend(q, q, rs, kl, t, 2 ** 40, 16),
               lambda: p.attend_prefix(q, q, i, 100, kl, t, 16), lambda: p.attend_prefix(q, q, i, -1, kl, t, 16), lambda: p.attend_prefix(q, q, i, 16, kl[:1], t, 16),
               lambda: p.append(x, x[:1], s), lambda: p.append(x[:, :64], x[:, :64], s), lambda: p.append(x, x, s[:1]), lambda: p.append(x, x, s.int()), lambda: p.append(x.t(), x.t(), s),
               lambda: serve.plan(ctx, 16, i, i[:2], t, i, i, i, i, s, i, i), lambda: serve.plan(ctx, 16, i[:2], i[:2], t, i, i, i[:2], i, s, i, i),
               lambda: serve.plan(ctx, 16, i[:2], i[:2], t, i, i, i, i, s, i[:1], i), lambda: serve.plan(ctx, 16, i[:2], i[:2], t, i, i, i, i, s, i, None),
               lambda: serve.penalize(ctx, lg, lg[:, :39]), lambda: serve.penalize(ctx, lg, lg, token=i), lambda: serve.penalize(ctx, lg, lg, history=torch.zeros(2, 3, dtype=torch.int64, device="cuda")),
               lambda: serve.penalize(ctx, lg, lg, repetition=f[:1]), lambda: serve.penalize(ctx, lg, lg, bias_ids=i32([[1], [2]]), bias=f), lambda: serve.penalize(ctx, lg, lg, mask=i32([[1], [1]])),
               lambda: serve.penalize(ctx, lg, lg, mask=i32([[1, 1]])), lambda: serve.penalize(ctx, lg, lg, repetition=[1.0, 1.0])]
    for n, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {n} was taken")
    for call in (lambda: p.attend(q.bfloat16(), q.bfloat16(), rs, kl, t, 1, 16), lambda: p.append(x.double(), x.double(), s), lambda: serve.penalize(ctx, lg.double(), lg),
                 lambda: serve.Pages(ctx, k.float(), v.float())):
        with pytest.raises(T.TcbError) as e:
            call()
        assert e.value.code == 2  # TCB_ERR_DTYPE
    with pytest.raises(TypeError):
        p.attend(q, q, rs, kl, t, "1", 16)


# ------------------------------------------------------------ pools

def pools(n_pages, KVH, page, hd, dtype, layout="heads", fill=math.nan):
    """Two pools seen as [pages, heads, positions, hd], in one of three memory orders."""
    if layout == "heads":
        k, v = (torch.full((n_pages, KVH, page, hd), fill, dtype=dtype, device="cuda") for _ in range(2))
    elif layout == "positions":
        k, v = (torch.full((n_pages, page, KVH, hd), fill, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
    else:  # K and V of a page side by side, padded
        both = torch.full((n_pages, 2, KVH, page, hd + 8), fill, dtype=dtype, device="cuda")[..., :hd]
        k, v = both[:, 0], both[:, 1]
    return k, v


def page_tables(lens, page, extra, r, first=0):
    n = [-(-x // page) for x in lens]
    ids = list(range(first, first + sum(n) + extra))
    r.shuffle(ids)
    width = max(n + [1]) + 1
    return [[ids.pop() if j < m else -1 for j in range(width)] for m in n]


def put(pool, table, rows, page, start=0):
    """rows [n, KVH, hd] into a request's pages from position start on"""
    if not rows.shape[0]:
        return
    p = torch.arange(start, start + rows.shape[0], device="cuda")
    g = torch.tensor(table, device="cuda")[p // page]
    pool.transpose(1, 2)[g, p % page] = rows.to(pool.dtype)


@pytest.mark.parametrize("xt", [F32, F16, BF16])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("layout", ["heads", "positions", "both"])
@pytest.mark.parametrize("T_,KVH,hd,page,skew", [(1, 1, 64, 16, 0), (5, 8, 128, 64, 0), (300, 2, 64, 256, 1), (77, 3, 128, 32, 1)])
def test_append(ctx, xt, dt, layout, T_, KVH, hd, page, skew):
    torch.manual_seed(T_)
    n_pages = -(-T_ // page) + 2
    k, v = pools(n_pages, KVH, page, hd, dt, layout, fill=7.0)
    wide = torch.randn(T_, 2 * KVH * hd + 8, device="cuda") * torch.logspace(-6, 4, T_, device="cuda")[:, None]
    wide = wide.to(xt)
    kr, vr = wide[:, skew:skew + KVH * hd], wide[:, KVH * hd + skew:2 * KVH * hd + skew]  # skew 1: rows off 16-byte alignment
    if page == 64:
        vr = vr.contiguous()  # rows of another stride
    slots = torch.randperm(n_pages * page, device="cuda")[:T_]
    if T_ > 4:
        slots[1] = -1
        slots[T_ - 1] = -5
    want_k, want_v = k.clone(), v.clone()
    keep = slots >= 0
    for w, x in ((want_k, kr), (want_v, vr)):
        w.transpose(1, 2)[slots[keep] // page, slots[keep] % page] = x[keep].view(-1, KVH, hd).to(dt)
    serve.Pages(ctx, k, v).append(kr, vr, slots)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_append_slot_outside_the_pools(ctx):
    k, v = pools(2, 2, 16, 64, F16, fill=3.0)
    x = torch.ones(2, 128, device="cuda")
    serve.Pages(ctx, k, v).append(x, x, torch.tensor([32, 5], device="cuda"))
    assert ctx.device_error(clear=True) == BOUNDS
    assert (k[0, :, 5] == 1).all() and (k == 3).sum() == k.numel() - 128


# ------------------------------------------------------------ attention

def attn_case(lens, rows, H, KVH, hd, page, dtype, layout="heads", seed=0, gain=2.0):
    """A cache that holds NaN wherever no request has a position, and rows of q."""
    r = random.Random(seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    tables = page_tables(lens, page, 3, r)
    k, v = pools(sum(-(-x // page) for x in lens) + 3, KVH, page, hd, dtype, layout)
    kv = []
    for n, t in zip(lens, tables):
        kr, vr = (torch.randn(n, KVH, hd, generator=g, device="cuda").to(dtype) for _ in range(2))
        put(k, t, kr, page)
        put(v, t, vr, page)
        kv.append((kr.double(), vr.double()))
    T_ = sum(rows)
    q = (gain * torch.randn(T_, H, hd, generator=g, device="cuda")).to(dtype)
    start = [0]
    for m in rows:
        start.append(start[-1] + m)
    return dict(k=k, v=v, kv=kv, q=q, tables=i32(tables), row_start=i32(start), kv_len=i32(lens), start=start)


def check_rows(out, c, lens, rows, dtype, window, sinks, scale, what):
    for b, (n, m) in enumerate(zip(lens, rows)):
        r0 = c["start"][b]
        pos = [n - m + i for i in range(m)]
        want, mag = R.attention(c["q"][r0:r0 + m].double(), *c["kv"][b], pos, scale, window, sinks)
        bound = R.attention_bound(want, mag, n, dtype)
        err = (out[r0:r0 + m].double() - want).abs()
        assert not torch.isnan(err).any(), f"{what}: NaN in request {b}"
        assert (err <= bound).all(), f"{what}: request {b} (len {n}, rows {m}): {(err / bound.clamp(min=1e-30)).max().item():.3g} of the bound"
        for i, p in enumerate(pos):
            if p < 0 or (window == 0 and sinks == 0):
                assert (out[r0 + i] == 0).all(), f"{what}: row {i} of request {b} sees nothing"


MASKS = [(None, 0), (1, 0), (16, 3), (37, 0), (100, 17), (4, 64), (0, 5), (0, 0), (100000, 2)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("H,KVH,hd,page,layout", [(8, 2, 128, 16, "heads"), (3, 3, 64, 64, "positions"), (16, 1, 128, 32, "both"),
                                                   (14, 2, 64, 256, "heads"), (40, 2, 128, 128, "positions"), (9, 3, 64, 16, "both")])
def test_attend_single_rows(ctx, dtype, window, sinks, H, KVH, hd, page, layout):
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 130, 257, 700]
    rows = [1] * len(lens)
    c = attn_case(lens, rows, H, KVH, hd, page, dtype, layout, seed=H + hd)
    out = torch.full_like(c["q"], math.nan)
    p = serve.Pages(ctx, c["k"], c["v"])
    p.attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], 1, 700, window=window, sinks=sinks)
    check_rows(out, c, lens, rows, dtype, window, sinks, 1 / math.sqrt(hd), "decode")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("H,KVH,hd,page,layout", [(8, 2, 128, 16, "heads"), (3, 3, 64, 64, "positions"), (16, 1, 128, 32, "both"),
                                                   (14, 2, 64, 256, "heads"), (40, 2, 128, 128, "positions")])
def test_attend_ragged_rows(ctx, dtype, window, sinks, H, KVH, hd, page, layout):
    lens = [1, 0, 3, 16, 33, 64, 150, 260, 300]
    rows = [1, 2, 5, 16, 2, 30, 0, 129, 3]  # requests 1 and 2 have rows before position 0
    c = attn_case(lens, rows, H, KVH, hd, page, dtype, layout, seed=H + hd + 1)
    out = torch.full_like(c["q"], math.nan)
    p = serve.Pages(ctx, c["k"], c["v"])
    p.attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], 129, 300, window=window, sinks=sinks)
    check_rows(out, c, lens, rows, dtype, window, sinks, 1 / math.sqrt(hd), "rows")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (37, 0), (100, 17), (4, 64), (0, 5), (0, 0)])
@pytest.mark.parametrize("H,KVH,hd,page,layout", [(8, 2, 128, 16, "heads"), (6, 6, 64, 64, "positions"), (16, 1, 128, 32, "both"),
                                                   (28, 4, 64, 256, "heads"), (40, 2, 128, 128, "positions")])
def test_attend_by_tiles(ctx, dtype, window, sinks, H, KVH, hd, page, layout):
    """The same through the tiles of many rows: max_rows and max_len only bound
    what the requests have, and bounds this large keep the rows together."""
    lens = [1, 0, 3, 16, 33, 64, 150, 260, 300]
    rows = [1, 2, 5, 16, 2, 30, 0, 129, 3]
    c = attn_case(lens, rows, H, KVH, hd, page, dtype, layout, seed=H + hd + 2)
    out = torch.full_like(c["q"], math.nan)
    serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], 188, 70000, window=window, sinks=sinks)
    check_rows(out, c, lens, rows, dtype, window, sinks, 1 / math.sqrt(hd), "tiles")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (37, 0), (4, 64), (0, 0)])
@pytest.mark.parametrize("H,KVH,hd,page", [(8, 2, 128, 16), (5, 1, 64, 64), (2, 2, 64, 32)])
def test_attend_few_long_among_many(ctx, dtype, window, sinks, H, KVH, hd, page):
    """Single rows, requests without rows and a few prompts: far fewer tiles
    than the longest request's for every request."""
    B = 300
    rows = [(1, 1, 0, 2)[b % 4] for b in range(B)]
    for b, m in ((5, 260), (127, 130), (128, 300), (129, 1), (299, 515)):
        rows[b] = m
    lens = [max(m, 3 + 7 * b % 90) for b, m in enumerate(rows)]
    c = attn_case(lens, rows, H, KVH, hd, page, dtype, seed=H + hd + 3)
    out = torch.full_like(c["q"], math.nan)
    serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], 600, 70000, window=window, sinks=sinks)
    check_rows(out, c, lens, rows, dtype, window, sinks, 1 / math.sqrt(hd), "among many")
    assert ctx.device_error(clear=True) == 0


@pytest.mark.parametrize("H,KVH,hd", [(1, 1, 64), (4, 1, 128)])
def test_attend_few_requests_with_rows(ctx, H, KVH, hd):
    """Most requests without rows, the positions of the others in parts."""
    rows, lens = [0] * 40, [50] * 40
    rows[3], rows[39], lens[3], lens[39] = 300, 5, 700, 1000
    c = attn_case(lens, rows, H, KVH, hd, 16, BF16, seed=hd)
    out = torch.full_like(c["q"], math.nan)
    serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], 1000, 70000)
    check_rows(out, c, lens, rows, BF16, None, 0, 1 / math.sqrt(hd), "few with rows")
    # lengths of requests without rows are looked at too, and row starts that fall
    p, bad = serve.Pages(ctx, c["k"], c["v"]), c["kv_len"].clone()
    bad[7] = -1
    p.attend(c["q"], out, c["row_start"], bad, c["tables"], 1000, 70000)
    assert ctx.device_error(clear=True) == BOUNDS
    check_rows(out, c, lens, rows, BF16, None, 0, 1 / math.sqrt(hd), "few with rows")
    falls = c["row_start"].clone()
    falls[20] = 0
    p.attend(c["q"], out, falls, c["kv_len"], c["tables"], 1000, 70000)
    assert ctx.device_error(clear=True) == BOUNDS


@pytest.mark.parametrize("H,KVH,hd", [(1, 1, 64), (2, 1, 128), (4, 1, 64), (8, 2, 64)])
def test_attend_one_prompt_among_requests_without_rows(ctx, H, KVH, hd):
    """Few tiles, found by count, and the positions in parts."""
    rows, lens = [0] * 40, [50] * 40
    rows[3], rows[39], lens[3], lens[39] = 1990, 5, 2100, 1000
    c = attn_case(lens, rows, H, KVH, hd, 16, F16, seed=hd + 1)
    p, out = serve.Pages(ctx, c["k"], c["v"]), torch.full_like(c["q"], math.nan)
    p.attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], 1995, 70000)
    check_rows(out, c, lens, rows, F16, None, 0, 1 / math.sqrt(hd), "one prompt")
    bad, falls = c["kv_len"].clone(), c["row_start"].clone()
    bad[7], falls[20] = -1, 0
    for start, n in ((c["row_start"], bad), (falls, c["kv_len"])):
        assert ctx.device_error(clear=True) == 0
        p.attend(c["q"], out, start, n, c["tables"], 1995, 70000)
        assert ctx.device_error(clear=True) == BOUNDS


def test_attend_row_starts_that_fall_single_rows(ctx):
    c = attn_case([9, 9, 9], [1, 1, 1], 4, 2, 64, 16, F16)
    serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], torch.empty_like(c["q"]), i32([0, 2, 1, 2]), c["kv_len"], c["tables"], 2, 9)
    assert ctx.device_error(clear=True) == BOUNDS


@pytest.mark.parametrize("rows,n", [([1], 5000), ([1], 4097), ([2], 3000), ([200], 2100), ([517], 517), ([1030], 1500)])
@pytest.mark.parametrize("dtype,H,KVH,hd", [(F16, 4, 1, 128), (BF16, 6, 2, 64)])
def test_attend_longer(ctx, rows, n, dtype, H, KVH, hd):
    """A sample of the rows of longer calls, with large scores that move the running maximum."""
    c = attn_case([n], rows, H, KVH, hd, 64, dtype, seed=n, gain=6.0)
    for window, sinks in ((None, 0), (700, 5)):
        out = torch.full_like(c["q"], math.nan)
        serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], rows[0], n, window=window, sinks=sinks, scale=0.2)
        at = sorted({0, 1, rows[0] // 3, rows[0] // 2, rows[0] - 2, rows[0] - 1} & set(range(rows[0])))
        pos = [n - rows[0] + i for i in at]
        want, mag = R.attention(c["q"][at].double(), *c["kv"][0], pos, 0.2, window, sinks)
        err = (out[at].double() - want).abs()
        assert (err <= R.attention_bound(want, mag, n, dtype)).all()
        assert torch.isfinite(out).all()


def test_attend_growing_and_falling_scores(ctx):
    """Keys whose scores rise along the sequence (every tile moves the
    maximum) and fall (none does), far apart enough to underflow."""
    n, hd = 640, 128
    for sign in (1.0, -1.0):
        c = attn_case([n, n], [1, 64], 2, 1, hd, 16, BF16, seed=3)
        q = torch.zeros(65, 2, hd, device="cuda")
        q[:, :, 0] = 8.0
        c["q"] = q.to(BF16)
        for b in range(2):
            kr = torch.zeros(n, 1, hd, device="cuda", dtype=BF16)
            kr[:, 0, 0] = (sign * torch.arange(n, device="cuda") * 0.25).to(BF16)
            put(c["k"], c["tables"][b].tolist(), kr, 16)
            c["kv"][b] = (kr.double(), c["kv"][b][1])
        out = torch.empty_like(c["q"])
        for m, rows in ((64, [1, 64]),):
            serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], m, n, scale=1.0)
            check_rows(out, c, [n, n], rows, BF16, None, 0, 1.0, "monotone scores")


@pytest.mark.parametrize("most", [200, 1 << 20])  # row by row, by tiles
@pytest.mark.parametrize("rows", [1, 3, 64])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attend_nonfinite_where_nothing_looks(ctx, rows, bad, most):
    """Non-finite K and V at cached positions outside the window of the last
    rows (and visible to none, or to the first rows only): rows that do not see
    them are unaffected; rows that see them are not finite."""
    n, H, KVH, hd, page, window, sinks = 200, 4, 2, 128, 16, 70, 3
    c = attn_case([n], [rows], H, KVH, hd, page, F16, seed=rows)
    first_lo = n - rows - window + 1  # the first row's window starts here
    spots = [sinks, first_lo - 1, 40] + ([first_lo] if rows > 1 else [])
    clean_k, clean_v = c["kv"][0]
    for name in ("k", "v"):
        for p in spots:
            c[name][c["tables"][0, p // page].item(), :, p % page] = bad
    out = torch.empty_like(c["q"])
    serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], rows if most == n else most, most,
                                            window=window, sinks=sinks)
    at = list(range(1 if rows > 1 else 0, rows))
    want, mag = R.attention(c["q"][at].double(), clean_k, clean_v, [n - rows + i for i in at], 1 / math.sqrt(hd), window, sinks)
    assert ((out[at].double() - want).abs() <= R.attention_bound(want, mag, n, F16)).all()
    if rows > 1 and bad == math.nan:
        assert torch.isnan(out[0]).all()


@pytest.mark.parametrize("most", [100, 1 << 20])
@pytest.mark.parametrize("rows", [2, 40])
def test_attend_nonfinite_after_a_row(ctx, rows, most):
    """A later position's V is infinite: rows before it do not see it."""
    n, hd = 100, 64
    c = attn_case([n], [rows], 2, 2, hd, 16, BF16, seed=rows)
    c["v"][c["tables"][0, (n - 1) // 16].item(), :, (n - 1) % 16] = math.inf
    out = torch.empty_like(c["q"])
    serve.Pages(ctx, c["k"], c["v"]).attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], rows, most)
    at = list(range(rows - 1))
    want, mag = R.attention(c["q"][at].double(), *c["kv"][0], [n - rows + i for i in at], 1 / math.sqrt(hd))
    assert ((out[at].double() - want).abs() <= R.attention_bound(want, mag, n, BF16)).all()
    assert not torch.isfinite(out[rows - 1]).any()


@pytest.mark.parametrize("rows,most", [(1, 90), (20, 90), (20, 1 << 20)])
def test_attend_strided_rows_and_untouched_ones(ctx, rows, most):
    """q as a part of wider rows, out likewise; rows outside every request keep what they hold."""
    lens, m = [50, 90], [rows, rows]
    c = attn_case(lens, m, 4, 2, 64, 32, F16, seed=rows)
    wide = torch.full((2 * rows + 3, 8 * 64), 5.0, dtype=F16, device="cuda")
    q = wide.view(-1, 8, 64)[:, 2:6]
    q[:2 * rows] = c["q"]
    res = torch.full((2 * rows + 3, 6 * 64), 9.0, dtype=F16, device="cuda")
    out = res.view(-1, 6, 64)[:, 1:5]
    serve.Pages(ctx, c["k"], c["v"]).attend(q, out, c["row_start"], c["kv_len"], c["tables"], rows, most)
    check_rows(out, c, lens, m, F16, None, 0, 1 / 8, "strided")
    assert (out[2 * rows:] == 9).all() and (res.view(-1, 6, 64)[:, 0] == 9).all() and (res.view(-1, 6, 64)[:, 5] == 9).all()


@pytest.mark.parametrize("rows,most", [(1, 64), (24, 64), (24, 1 << 20)])
def test_attend_device_findings(ctx, rows, most):
    """A page outside the pools, a length past max_len or the table, and more
    rows than max_rows are reported, and the other requests are right."""
    lens, m = [40, 64, 33], [rows, rows, rows]
    c = attn_case(lens, m, 4, 2, 128, 16, BF16, seed=rows)
    p = serve.Pages(ctx, c["k"], c["v"])

    def go(tables=None, kv_len=None, row_start=None, max_rows=rows, max_len=most):
        out = torch.zeros_like(c["q"])
        p.attend(c["q"], out, c["row_start"] if row_start is None else row_start, c["kv_len"] if kv_len is None else kv_len,
                 c["tables"] if tables is None else tables, max_rows, max_len)
        return out

    for page in (-1, c["k"].shape[0], 2 ** 31 - 1, -2 ** 31):
        t = c["tables"].clone()
        t[1, 2] = page
        out = go(tables=t)
        assert ctx.device_error(clear=True) == BOUNDS
        for b in (0, 2):
            sub = {**c, "q": c["q"][b * rows:(b + 1) * rows], "kv": [c["kv"][b]], "start": [0]}
            check_rows(out[b * rows:(b + 1) * rows], sub, [lens[b]], [rows], BF16, None, 0, 1 / math.sqrt(128), "neighbour")
    for n in (65 if most == 64 else 16 * c["tables"].shape[1] + 1, 2 ** 31 - 1, -1):
        out = go(kv_len=i32([40, n, 33]))
        assert ctx.device_error(clear=True) == BOUNDS
        sub = {**c, "q": c["q"][:rows], "kv": [c["kv"][0]], "start": [0]}
        check_rows(out[:rows], sub, [40], [rows], BF16, None, 0, 1 / math.sqrt(128), "neighbour")
    go(kv_len=i32([40, 16 * c["tables"].shape[1] + 1, 33]), max_len=1 << 20)
    assert ctx.device_error(clear=True) == BOUNDS
    go(row_start=i32([0, -5, 2 ** 31 - 1, 7]))  # held to the rows of q
    ctx.device_error(clear=True)
    if rows > 1:
        go(max_rows=rows - 1)
        assert ctx.device_error(clear=True) == BOUNDS


@pytest.mark.parametrize("rows,most", [(1, 200), (3, 200), (70, 1 << 20)])
def test_attend_offsets_past_32_bits(ctx, rows, most):
    """Pages whose elements lie past 2^31 and 2^32 of the pool (K and V in one
    array; only the pages in use are written)."""
    KVH, page, hd = 2, 64, 128
    stride = KVH * page * hd
    n_pages = (2 ** 32) // stride + 40
    if torch.cuda.mem_get_info()[0] < 2 * n_pages * stride + (4 << 30):
        pytest.skip("9 GB of device memory are needed")
    pool = torch.empty((n_pages, KVH, page, hd), dtype=BF16, device="cuda")
    n = 200
    table = [n_pages - 1, 3, 2 ** 31 // stride + 1, n_pages - 20]
    x = torch.randn(n, KVH, hd, device="cuda").to(BF16)
    put(pool, table, x, page)
    c = dict(q=torch.randn(rows, 4, hd, device="cuda").to(BF16), kv=[(x.double(), x.double())], start=[0])
    out = torch.empty_like(c["q"])
    p = serve.Pages(ctx, pool, pool)
    p.attend(c["q"], out, i32([0, rows]), i32([n]), i32([table]), rows, most)
    check_rows(out, c, [n], [rows], BF16, None, 0, 1 / math.sqrt(hd), "far pages")
    # and the append finds them
    y = torch.randn(1, KVH * hd, device="cuda")
    p.append(y, y, torch.tensor([(n_pages - 1) * page + 5], device="cuda"))
    assert torch.equal(pool[n_pages - 1, :, 5], y.view(KVH, hd).to(BF16))


@pytest.mark.parametrize("rows,most", [(1, 1000), (33, 1000), (33, 1 << 20)])
def test_attend_again_is_the_same_bits(ctx, rows, most):
    lens = [500, 3, 64, 1000]
    m = [min(rows, n) for n in lens]
    c = attn_case(lens, m, 8, 2, 128, 16, F16, seed=1)
    p, outs = serve.Pages(ctx, c["k"], c["v"]), []
    for _ in range(3):
        out = torch.full_like(c["q"], math.nan)
        p.attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], rows, most)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_attend_on_a_side_stream_and_in_a_graph(ctx):
    c = attn_case([300, 40], [1, 1], 8, 2, 128, 16, F16, seed=2)
    p = serve.Pages(ctx, c["k"], c["v"])
    want, out = torch.empty_like(c["q"]), torch.zeros_like(c["q"])
    p.attend(c["q"], want, c["row_start"], c["kv_len"], c["tables"], 1, 300, window=100, sinks=4)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    p.attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], 1, 300, window=100, sinks=4, stream=s)
    s.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.attend(c["q"], out, c["row_start"], c["kv_len"], c["tables"], 1, 300, window=100, sinks=4)
    c["kv_len"].copy_(i32([299, 39]))  # lengths are read on the device
    g.replay()
    p.attend(c["q"], want, c["row_start"], c["kv_len"], c["tables"], 1, 300, window=100, sinks=4)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_captured_graphs_outlive_larger_calls():
    """A graph names the scratch of its capture; a later call that needs more
    leaves it in place."""
    own = T.Context(0)
    c = attn_case([3000], [1], 4, 1, 128, 64, F16, seed=5)
    p = serve.Pages(own, c["k"], c["v"])
    args = (c["row_start"], c["kv_len"], c["tables"], 1, 3000)
    want, out = torch.empty_like(c["q"]), torch.zeros_like(c["q"])
    p.attend(c["q"], want, *args)  # several clusters: joined through scratch and counters
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.attend(c["q"], out, *args)
    d = attn_case([400] * 6, [200] * 6, 4, 1, 128, 64, F16, seed=6)
    big = torch.empty_like(d["q"])
    serve.Pages(own, d["k"], d["v"]).attend(d["q"], big, d["row_start"], d["kv_len"], d["tables"], 200, 1 << 20)
    run_logits(own, logits_case(3000, 40, 0, seed=1))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and own.device_error() == 0


# ------------------------------------------------------------ shared prefix

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,P,H,KVH,hd,page,layout", [
    (1, 1, 4, 2, 128, 16, "heads"), (3, 15, 4, 1, 64, 16, "positions"), (5, 16, 8, 2, 128, 16, "both"), (9, 17, 6, 3, 64, 32, "heads"),
    (4, 300, 32, 8, 128, 64, "heads"), (33, 511, 16, 2, 128, 16, "positions"), (64, 130, 8, 8, 64, 256, "heads"), (40, 640, 32, 1, 128, 128, "both"),
    (17, 0, 8, 2, 128, 16, "heads"), (7, 2100, 14, 2, 64, 16, "heads"),
    # read once for all requests from here on
    (64, 1111, 16, 8, 128, 16, "heads"), (61, 777, 32, 4, 128, 64, "positions"), (33, 2049, 24, 8, 64, 256, "both"), (5, 9000, 8, 2, 128, 32, "heads"),
    (64, 4100, 20, 1, 128, 128, "heads"), (48, 900, 7, 7, 128, 16, "positions")])
def test_attend_prefix(ctx, dtype, B, P, H, KVH, hd, page, layout):
    r = random.Random(P + B)
    lens = [P + r.choice([0, 1, 2, 15, 16, 17, 100, 200]) for _ in range(B)]
    lens[0] = P + 1
    if B > 4:
        lens[1], lens[2], lens[3] = 0, P // 2, min(P, 1)
    first = -(-P // page)
    whole = P // page
    sub = page_tables([max(0, n - whole * page) for n in lens], page, 2, r, first)
    tables = [[-1] * whole + t for t in sub]
    prefix = list(range(first))
    r.shuffle(prefix)
    n_pages = max(max(t) for t in tables + [[first]]) + 3
    k, v = pools(n_pages, KVH, page, hd, dtype, layout)
    torch.manual_seed(B)
    pk, pv = (torch.randn(P, KVH, hd, device="cuda").to(dtype) for _ in range(2))
    put(k, prefix, pk, page)
    put(v, prefix, pv, page)
    kv = []
    for n, t in zip(lens, tables):
        sk, sv = (torch.randn(max(0, n - P), KVH, hd, device="cuda").to(dtype) for _ in range(2))
        put(k, t, sk, page, P)
        put(v, t, sv, page, P)
        kv.append((torch.cat([pk, sk]).double(), torch.cat([pv, sv]).double()))
    q = (2 * torch.randn(B, H, hd, device="cuda")).to(dtype)
    out = torch.full_like(q, math.nan)
    serve.Pages(ctx, k, v).attend_prefix(q, out, i32(prefix), P, i32(lens), i32(tables), max(lens))
    for b, n in enumerate(lens):
        want, mag = R.attention(q[b:b + 1].double(), *kv[b], [n - 1], 1 / math.sqrt(hd))
        err = (out[b:b + 1].double() - want).abs()
        assert (err <= R.attention_bound(want, mag, n, dtype)).all(), (b, n)
        if n == 0:
            assert (out[b] == 0).all()


@pytest.mark.parametrize("P,B", [(100, 3), (2300, 63)])
def test_attend_prefix_nonfinite_tail_of_the_prefix(ctx, P, B):
    """Requests shorter than the prefix do not see its later positions."""
    page, hd, KVH = 16, 128, 1 if P == 100 else 2
    n = -(-P // page)
    k, v = pools(n + 2, KVH, page, hd, F16)
    x = torch.randn(P, KVH, hd, device="cuda").half()
    y = x.clone()
    y[60:] = math.inf
    put(k, list(range(n)), x, page)
    put(v, list(range(n)), y, page)
    q = torch.randn(B, 4, hd, device="cuda").half()
    out = torch.empty_like(q)
    lens = [60, P, 31] + [P] * (B - 3)
    serve.Pages(ctx, k, v).attend_prefix(q, out, i32(list(range(n))), P, i32(lens), i32([[-1] * n] * B), P)
    for b in (0, 2):
        want, mag = R.attention(q[b:b + 1].double(), x.double(), x.double(), [lens[b] - 1], 1 / math.sqrt(hd))
        assert ((out[b:b + 1].double() - want).abs() <= R.attention_bound(want, mag, P, F16)).all()
    assert not torch.isfinite(out[1]).any() and not torch.isfinite(out[3:]).any()


def test_attend_prefix_device_findings(ctx):
    k, v = pools(4, 1, 16, 64, F16, fill=0.0)
    q = torch.randn(2, 2, 64, device="cuda").half()
    out = torch.empty_like(q)
    p = serve.Pages(ctx, k, v)
    many = torch.randn(64, 2, 64, device="cuda").half()  # read once for all
    pages = [0, 1, 2] * 1000
    pages[1500] = 4
    p.attend_prefix(many, torch.empty_like(many), i32(pages), 48000, i32([48000] * 64), i32([[-1] * 3000] * 64), 48000)
    assert ctx.device_error(clear=True) == BOUNDS
    p.attend_prefix(q, out, i32([0, 99]), 32, i32([32, 32]), i32([[-1, -1, 2]] * 2), 40)
    assert ctx.device_error(clear=True) == BOUNDS
    p.attend_prefix(q, out, i32([0, 1]), 32, i32([33, 41]), i32([[-1, -1, 2]] * 2), 40)
    assert ctx.device_error(clear=True) == BOUNDS


# ------------------------------------------------------------ logits

def logits_case(B, V, width, seed, n_bias=0, n_masks=0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    c = dict(logits=(3 * torch.randn(B, V, generator=g)).to(dtype), history=torch.randint(0, V, (B, max(width, 1)), generator=g)[:, :width],
             total_len=[r.randint(0, width) for _ in range(B)], repetition=1 + torch.rand(B, generator=g), frequency=torch.rand(B, generator=g) - 0.3,
             presence=torch.rand(B, generator=g) - 0.3)
    c["total_len"][0] = width
    c["prompt_len"] = [r.randint(0, n) for n in c["total_len"]]
    if width:
        c["history"][:, ::3] = c["history"][:, :1].clone()  # repeats
        c["history"][-1, -1] = -1  # an unused entry
        c["history"][0, width // 2] = V + 7
    if n_bias:
        c["bias_ids"] = torch.randint(-1, V, (B, n_bias), generator=g).int()
        c["bias_ids"][:, -1] = c["bias_ids"][:, 0]  # the last of two entries for a token counts
        c["bias"] = 2 * torch.randn(B, n_bias, generator=g)
    if n_masks:
        c["mask"] = torch.randint(-2 ** 31, 2 ** 31, (n_masks, -(-V // 32)), generator=g).int()
        c["mask_row"] = [r.randrange(-1, n_masks) for _ in range(B)]
    return c


def run_logits(ctx, c, out_dtype=F32, inplace=False, stride=0):
    dev = {k: (i32(v) if isinstance(v, list) else v.cuda()) for k, v in c.items()}
    x = dev.pop("logits")
    if stride:
        x = torch.nn.functional.pad(x, (0, stride))[:, :x.shape[1]]
    out = x if inplace else torch.full(x.shape, 77.0, dtype=out_dtype, device="cuda")
    token = torch.full((x.shape[0],), -9, dtype=torch.int64, device="cuda")
    serve.penalize(ctx, x, out, token, **dev)
    return out, token


def check_logits(c, out, token):
    B, V = c["logits"].shape
    for b in range(B):
        allowed = None
        if "mask" in c and c["mask_row"][b] >= 0:
            w = c["mask"][c["mask_row"][b]].long()
            allowed = ((w[:, None] >> torch.arange(32)) & 1).view(-1)[:V].bool()
        bias = list(zip(c["bias_ids"][b].tolist(), c["bias"][b].double().tolist())) if "bias" in c else []
        total = c["total_len"][b] if "history" in c else 0
        prompt = c["prompt_len"][b] if "prompt_len" in c else 0
        hist = c["history"][b].tolist() if "history" in c else []
        x = c["logits"][b].double()
        want = R.penalties(x, hist, prompt, total, c["repetition"][b].double().item() if "repetition" in c else 1.0,
                           c["frequency"][b].double().item() if "frequency" in c else 0.0, c["presence"][b].double().item() if "presence" in c else 0.0, bias, allowed)
        got = out[b].cpu()
        # at most five roundings to f32 of values no larger than the sum of magnitudes, then one to the output's type
        size = x.abs() * 2 + (total + 2) * 1.3 + sum(abs(v) for _, v in bias)
        size = torch.where(want == x, x.abs(), size)
        u = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}[got.dtype]
        fin = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), fin) and torch.equal(got[~fin].double(), want[~fin])
        err = (got.double() - want).abs()[fin]
        assert (err <= (5 * 2.0 ** -24 * size + u * want.abs() + (2.0 ** -25 if got.dtype == F16 else 0))[fin]).all(), b
        if got.dtype == F32 and token is not None:
            top = got.max()
            first = int((got == top).nonzero()[0]) if top > -math.inf else -1
            assert token[b].item() == first, b


@pytest.mark.parametrize("B,V,width,n_bias,n_masks", [(1, 1, 0, 0, 0), (1, 31, 5, 1, 1), (3, 33, 40, 4, 2), (2, 1000, 300, 0, 0), (5, 4095, 64, 7, 3),
                                                      (4, 4097, 1, 300, 0), (2, 128256, 3000, 50, 2), (70, 513, 20, 3, 5)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_penalize(ctx, B, V, width, n_bias, n_masks, dtype):
    c = logits_case(B, V, width, seed=V + B, n_bias=n_bias, n_masks=n_masks, dtype=dtype)
    check_logits(c, *run_logits(ctx, c))
    check_logits(c, *run_logits(ctx, c, stride=3))
    check_logits(c, *run_logits(ctx, c, out_dtype=dtype, inplace=True))


@pytest.mark.parametrize("drop", ["history", "repetition", "frequency", "presence", "prompt_len", "mask_row", "bias"])
def test_penalize_parts_left_out(ctx, drop):
    c = logits_case(3, 700, 50, seed=4, n_bias=6, n_masks=3)
    gone = {"history": ("history", "prompt_len", "total_len"), "bias": ("bias", "bias_ids")}.get(drop, (drop,))
    d = {k: v for k, v in c.items() if k not in gone}
    out, token = run_logits(ctx, d)
    check_logits({**d, "mask_row": c["mask_row"] if "mask_row" in d else [0, 1, 2]}, out, token)


def test_penalize_ties_nan_and_nothing_allowed(ctx):
    V = 9000
    x = torch.zeros(6, V)
    x[0, [17, 5000, 8999]] = 4.0  # equal maxima: the lowest token
    x[1] = -math.inf
    x[2, 5] = math.nan
    x[2, 8000] = 1.0
    x[3] = math.nan
    x[4] = -0.0
    x[4, 8998] = 0.0  # +0 and -0 are equal
    x[5, 4200] = math.inf
    mask = torch.zeros(1, -(-V // 32), dtype=torch.int32)
    out, token = run_logits(ctx, dict(logits=x))
    assert token.tolist() == [17, -1, 8000, -1, 0, 4200]
    assert torch.equal(out.cpu().view(torch.int32), x.view(torch.int32))
    out, token = run_logits(ctx, dict(logits=x, mask=mask, mask_row=[0, 0, 0, 0, -1, 0]))
    assert token.tolist() == [-1, -1, -1, -1, 0, -1] and (out[[0, 1, 2, 3, 5]] == -math.inf).all()
    mask[0, 8000 // 32] = 1 << (8000 % 32)
    out, token = run_logits(ctx, dict(logits=x, mask=mask, mask_row=[0] * 6))
    assert token.tolist() == [8000, -1, 8000, -1, 8000, 8000]


def test_penalize_lengths_past_the_history_and_a_mask_row_past_the_masks(ctx):
    c = logits_case(2, 300, 10, seed=9, n_masks=1)
    c["mask_row"] = [-1, -1]
    want, _ = run_logits(ctx, {**c, "total_len": [10, 10], "prompt_len": [3, 0]})
    got, _ = run_logits(ctx, {**c, "total_len": [10 ** 9, 10], "prompt_len": [3, -4]})
    assert torch.equal(want, got)
    got, _ = run_logits(ctx, {**c, "total_len": [-5, 0]})
    assert torch.equal(got.cpu(), c["logits"])
    run_logits(ctx, {**c, "mask_row": [0, 1]})
    assert ctx.device_error(clear=True) == BOUNDS


def test_penalize_counts_every_occurrence(ctx):
    """One token thousands of times: the count is whole."""
    h = torch.full((1, 70001), 3, dtype=torch.int64)
    c = dict(logits=torch.zeros(1, 50), history=h, prompt_len=[1], total_len=[70001], frequency=torch.tensor([0.5]))
    out, token = run_logits(ctx, c)
    assert out[0, 3].item() == -35000.0 and token.item() == 0
