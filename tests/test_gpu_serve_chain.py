"""Steps behind one another without a wait: every kernel reads what the ones
before it have just written."""
import math

import pytest
import torch

import tcb_b200 as T
from tcb_b200 import serve

import serve_ref as R
from test_gpu_serve import F16, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,P,H,KVH", [(61, 2304, 16, 4), (24, 8192, 8, 2), (4, 48, 8, 2)])
def test_steps_behind_a_prefix(B, P, H, KVH):
    """plan, append and attend_prefix of 24 steps queued at once; the lengths,
    table entries and K/V rows of a step are written right before its
    attention, the first positions of the prefix again at every step."""
    ctx, page, hd, steps = T.Context(0), 16, 128, 24
    first, width = P // page, P // page + 3
    n_pages = first + 3 * B
    k, v = (torch.full((n_pages, KVH, page, hd), math.nan, dtype=F16, device="cuda") for _ in "kv")
    torch.manual_seed(B)
    p = serve.Pages(ctx, k, v)
    prefix = torch.randperm(first, device="cuda").to(torch.int32)
    at = torch.arange(P, device="cuda")
    slots0 = prefix[at // page].long() * page + at % page
    pk, pv = (torch.randn(P, KVH * hd, device="cuda") for _ in "kv")
    p.append(pk, pv, slots0)
    tables = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    tables[:, :first] = prefix
    free = torch.arange(first, n_pages, dtype=torch.int32, device="cuda")
    n_free, cached, fresh = i32([3 * B]), torch.full((B,), P, dtype=torch.int32, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda")
    rs, kl, bal, taken = i32([0] * (B + 1)), i32([0] * B), i32([0]), i32([0])
    slots, pos = torch.zeros(B, dtype=torch.int64, device="cuda"), i32([0] * B)
    heads = [torch.randn(2, 40, KVH * hd, device="cuda") for _ in range(steps)]
    rows = [torch.randn(2, B, KVH * hd, device="cuda") for _ in range(steps)]
    qs = [torch.randn(B, H, hd, device="cuda").to(F16) * 2 for _ in range(steps)]
    outs = [torch.full_like(qs[0], math.nan) for _ in range(steps)]
    torch.cuda.synchronize()
    for s in range(steps):
        serve.plan(ctx, page, cached, fresh, tables, free, n_free, rs, kl, slots, pos, bal, taken)
        p.append(*heads[s], slots0[:40])
        p.append(*rows[s], slots)
        p.attend_prefix(qs[s], outs[s], prefix, P, kl, tables, P + steps)
        n_free.sub_(taken)
        cached.copy_(kl)
    torch.cuda.synchronize()
    assert ctx.device_error(clear=True) == 0
    half = lambda x: x.to(F16).double().view(-1, KVH, hd)
    kd, vd = half(pk), half(pv)
    for s in range(steps):
        for x, h in zip((kd, vd), heads[s]):
            x[:40] = half(h)
        sk, sv = (torch.stack([half(r[i]) for r in rows[:s + 1]], 1) for i in (0, 1))
        for b in range(0, B, max(1, B // 6)):
            n = P + s + 1
            want, mag = R.attention(qs[s][b:b + 1].double(), torch.cat([kd, sk[b]]), torch.cat([vd, sv[b]]), [n - 1], 1 / math.sqrt(hd))
            assert ((outs[s][b:b + 1].double() - want).abs() <= R.attention_bound(want, mag, n, F16)).all(), (s, b)
