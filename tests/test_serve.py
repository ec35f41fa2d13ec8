"""Refusals of the serving operators' C entry points and Python view, and the
plan's reference, without a GPU."""
import ctypes
import types

import pytest
import torch

import tcb_b200 as T
from tcb_b200 import serve

import serve_ref as R

NULL, DTYPE, SHAPE, ALIGN, UNSUPPORTED, TOO_LARGE = 1, 2, 3, 4, 8, 11


@pytest.fixture(scope="module")
def ctx():
    """An address that is never dereferenced: every call here is refused on its arguments."""
    buf = ctypes.create_string_buffer(4096)
    return buf


def pages(**kw):
    d = dict(k=0x1000, v=0x2000, dtype=T.F16, n_pages=4, page=16, n_kv_heads=2, head_dim=128, page_stride=4096,
             head_stride=2048, pos_stride=128)
    d.update(kw)
    return serve._KvPages(**d)


def attn(ctx, kv=None, **kw):
    d = dict(B=2, T=2, H=4, q=0x1000, ldq=512, out=0x2000, ldo=512, row_start=0x100, kv_len=0x200, tables=0x300,
             width=4, ldt=4, max_rows=1, max_len=64, scale=0.1, window=-1, sinks=0)
    d.update(kw)
    return serve._lib().tcb_page_attn(ctx, ctypes.byref(pages() if kv is None else kv), *d.values(), None)


def prefix(ctx, kv=None, **kw):
    d = dict(B=2, H=4, q=0x1000, ldq=512, out=0x2000, ldo=512, prefix=0x400, prefix_len=16, kv_len=0x200,
             tables=0x300, width=4, ldt=4, max_len=64, scale=0.1)
    d.update(kw)
    return serve._lib().tcb_prefix_attn(ctx, ctypes.byref(pages() if kv is None else kv), *d.values(), None)


def append(ctx, kv=None, **kw):
    d = dict(T=2, k=0x1000, ldk=256, v=0x2000, ldv=256, xdtype=T.F32, slots=0x100)
    d.update(kw)
    return serve._lib().tcb_kv_append(ctx, ctypes.byref(pages() if kv is None else kv), *d.values(), None)


def plan(ctx, **kw):
    d = dict(B=2, page=16, cached=0x100, fresh=0x200, tables=0x300, width=4, ldt=4, free=0x400, free_cap=8,
             n_free=0x500, rows=2, row_start=0x600, kv_len=0x700, slots=0x800, positions=0x900, balance=0xA00, taken=0)
    d.update(kw)
    return serve._lib().tcb_page_plan(ctx, *d.values(), None)


def logits(ctx, **kw):
    d = dict(B=2, V=100, logits=0x1000, dtype=T.F32, ld=100, out=0x2000, odtype=T.F32, ldo=100, token=0x100)
    d.update(kw)
    return serve._lib().tcb_logits_penalize(ctx, ctypes.byref(serve._LogitsArgs(**d)), None)


def test_null_context():
    assert [f(None) for f in (plan, append, attn, prefix, logits)] == [NULL] * 5


@pytest.mark.parametrize("bad,code", [
    (dict(k=0), NULL), (dict(v=None), NULL), (dict(dtype=T.F32), DTYPE), (dict(dtype=77), DTYPE), (dict(page=8), SHAPE),
    (dict(page=48), SHAPE), (dict(page=512), SHAPE), (dict(n_pages=0), SHAPE), (dict(head_dim=96), SHAPE),
    (dict(n_kv_heads=0), SHAPE), (dict(pos_stride=64), SHAPE), (dict(page_stride=4100), ALIGN),
    (dict(pos_stride=132), ALIGN), (dict(k=0x1008), ALIGN)])
def test_pools(ctx, bad, code):
    kv = pages(**bad)
    assert append(ctx, kv) == attn(ctx, kv) == prefix(ctx, kv) == code


@pytest.mark.parametrize("bad,code", [
    (dict(B=-1), SHAPE), (dict(T=-1), SHAPE), (dict(H=3), SHAPE), (dict(H=0), SHAPE), (dict(B=65536), SHAPE), (dict(ldq=511), SHAPE),
    (dict(ldo=8), SHAPE), (dict(ldt=3), SHAPE), (dict(width=-1), SHAPE), (dict(max_len=-1), SHAPE), (dict(max_rows=-1), SHAPE),
    (dict(sinks=-1), SHAPE), (dict(scale=float("nan")), SHAPE), (dict(scale=float("inf")), SHAPE), (dict(q=0), NULL), (dict(out=0), NULL),
    (dict(kv_len=0), NULL), (dict(tables=0), NULL), (dict(row_start=0), NULL), (dict(q=0x1008), ALIGN), (dict(out=0x1002), ALIGN),
    (dict(ldq=516), ALIGN), (dict(kv_len=0x202), ALIGN), (dict(tables=0x301), ALIGN), (dict(row_start=0x102), ALIGN),
    (dict(B=0), 0), (dict(T=0), 0), (dict(max_rows=0), 0)])
def test_attention(ctx, bad, code):
    assert attn(ctx, **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(B=-1), SHAPE), (dict(H=5), SHAPE), (dict(prefix_len=-1), SHAPE), (dict(prefix=0), NULL), (dict(prefix=0x402), ALIGN),
    (dict(q=0), NULL), (dict(scale=float("nan")), SHAPE), (dict(B=0), 0)])
def test_prefix_attention(ctx, bad, code):
    assert prefix(ctx, **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(T=-1), SHAPE), (dict(ldk=255), SHAPE), (dict(ldv=255), SHAPE), (dict(xdtype=T.Q4_K), DTYPE), (dict(k=0), NULL), (dict(slots=0), NULL),
    (dict(k=0x1002), ALIGN), (dict(slots=0x104), ALIGN), (dict(T=0), 0)])
def test_append(ctx, bad, code):
    assert append(ctx, **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(B=-1), SHAPE), (dict(page=17), SHAPE), (dict(width=-1), SHAPE), (dict(ldt=3), SHAPE), (dict(rows=-1), SHAPE), (dict(free_cap=-1), SHAPE),
    (dict(B=8193), TOO_LARGE), (dict(cached=0), NULL), (dict(fresh=0), NULL), (dict(tables=0), NULL),
    (dict(free=0), NULL), (dict(n_free=0), NULL), (dict(row_start=0), NULL), (dict(kv_len=0), NULL), (dict(slots=0), NULL),
    (dict(positions=0), NULL), (dict(balance=0), NULL), (dict(balance=0x500), UNSUPPORTED), (dict(taken=0x500), UNSUPPORTED), (dict(slots=0x804), ALIGN), (dict(cached=0x101), ALIGN)])
def test_plan(ctx, bad, code):
    assert plan(ctx, **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(B=-1), SHAPE), (dict(V=-1), SHAPE), (dict(B=65536), SHAPE), (dict(ld=99), SHAPE), (dict(ldo=99), SHAPE), (dict(dtype=T.Q4_K), DTYPE), (dict(odtype=3), DTYPE),
    (dict(logits=0), NULL), (dict(out=0), NULL), (dict(logits=0x1002), ALIGN), (dict(token=0x104), ALIGN),
    (dict(out=0x1000, odtype=T.F16), UNSUPPORTED), (dict(out=0x1000, ldo=104), UNSUPPORTED),
    (dict(history=0x100, hist_width=4, ldh=4), NULL), (dict(history=0x100, hist_width=4, ldh=3, total_len=0x100), SHAPE),
    (dict(history=0x104, hist_width=4, ldh=4, total_len=0x100), ALIGN), (dict(bias_ids=0x100, n_bias=3, ldb=3), NULL),
    (dict(bias_ids=0x100, bias=0x100, n_bias=3, ldb=2), SHAPE), (dict(mask=0x100, n_masks=2, ldm=3), SHAPE),
    (dict(mask=0x100, n_masks=0, ldm=4), SHAPE), (dict(mask=0x102, n_masks=1, ldm=4), ALIGN), (dict(B=0), 0), (dict(V=0), 0)])
def test_logits(ctx, bad, code):
    assert logits(ctx, **bad) == code


def test_python_view_refuses_host_tensors(ctx):
    c = types.SimpleNamespace(handle=ctypes.c_void_p(ctypes.addressof(ctx)), device=0)
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: serve.Pages(c, k, k), lambda: serve.Pages(c, k, k[:2]), lambda: serve.penalize(c, torch.zeros(2, 8), torch.zeros(2, 8)),
                 lambda: serve.plan(c, 16, i, i, i.view(2, 1), i, i, i, i, i.long(), i, i), lambda: serve.plan(c, 16, None, i, i, i, i, i, i, i, i, i)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        serve._view().plan(0)


def test_plan_reference():
    t, rs, kl, sl, ps, balance, taken = R.plan(16, [0, 15, 16, 40], [1, 2, 0, 100], [[-1, -1], [7, -1], [8, -1], [1, 2]], [3, 4, 5], 3, 120)
    assert t == [[5, -1], [7, 4], [8, -1], [1, 2]]
    assert rs == [0, 1, 3, 3, 103] and kl == [1, 17, 16, 0] and (balance, taken) == (1, 2)
    # a request that lacks no page is served behind one that is refused for want of pages
    assert R.plan(16, [0, 3], [40, 1], [[-1] * 3, [6, -1, -1]], [4, 5], 2, 41)[5:] == (-1, 0)
    assert sl[:4] == [80, 7 * 16 + 15, 4 * 16, -1] and ps[:4] == [0, 15, 16, -1]
