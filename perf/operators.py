"""Cases of the serving operators: the page plan of a step, the append of its
K/V rows into the paged cache, attention over the pages (a window and a few
first positions that stay visible), attention of a batch over one shared
prefix, and the penalties, biases and grammar masks on its logits.

own = False computes them with elementary torch operations in 32 bits;
own = True makes the calls of tcb_b200.serve.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
V_LLAMA = 128256  # the vocabulary of the framework's 8B and 70B configurations

_ctx = None


def _context():
    """The framework's context, made once as a program makes it (only where own is true)."""
    global _ctx
    if _ctx is None:
        import tcb_b200

        _ctx = tcb_b200.Context(0)
    return _ctx


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a decode step's page plan for 16 sequences (the batch of the 70B decode): one new position each
        {"name": "plan_decode_16", "op": "plan", "B": 16, "page": 16, "max_cached": 1152, "max_fresh": 1, "tight": False, "lens": 1},
        # admission of a queue of prompts: ragged chunks of a thousand requests, with too few free pages for the last ones
        {"name": "plan_prompts_1024", "op": "plan", "B": 1024, "page": 64, "max_cached": 8192, "max_fresh": 1024, "tight": True, "lens": 2},
        # a decode step's K/V rows of 16 sequences, from the f32 rows of the projections
        {"name": "append_decode_16", "op": "append", "T": 16, "KVH": 8, "hd": 128, "page": 16, "xtype": "f32", "dtype": "f16", "lens": 3},
        # the K/V rows of a full prompt pass of several sequences, padded rows among them
        {"name": "append_prompt_16k", "op": "append", "T": 16391, "KVH": 8, "hd": 128, "page": 64, "xtype": "bf16", "dtype": "bf16", "lens": 4},
        # one sequence's decode step at the 8B shape: latency
        {"name": "attn_decode_1", "op": "attn", "B": 1, "H": 32, "KVH": 8, "hd": 128, "page": 16, "dtype": "f16", "max_rows": 1, "max_len": 4001,
         "window": 1024, "sinks": 4, "lens": 5},
        # a serving batch's decode step at the 70B shape: ragged long caches, an idle slot among them
        {"name": "attn_decode_64", "op": "attn", "B": 64, "H": 64, "KVH": 8, "hd": 128, "page": 32, "dtype": "bf16", "max_rows": 1, "max_len": 32768,
         "window": 16384, "sinks": 16, "lens": 6},
        # chunks of prompts behind ragged caches at the 8B shape
        {"name": "attn_chunks_7", "op": "attn", "B": 7, "H": 32, "KVH": 8, "hd": 128, "page": 16, "dtype": "f16", "max_rows": 515, "max_len": 2311,
         "window": 512, "sinks": 8, "lens": 7},
        # one long prompt at the 8B shape
        {"name": "attn_prompt_8k", "op": "attn", "B": 1, "H": 32, "KVH": 8, "hd": 128, "page": 64, "dtype": "bf16", "max_rows": 8192, "max_len": 8192,
         "window": 4096, "sinks": 4, "lens": 8},
        # four answers to one prompt (the 8B batch of four)
        {"name": "prefix_4", "op": "prefix", "B": 4, "H": 32, "KVH": 8, "hd": 128, "page": 16, "dtype": "f16", "prefix": 509, "max_suffix": 128, "lens": 9},
        # a serving batch behind one long instruction text at the 70B shape
        {"name": "prefix_64", "op": "prefix", "B": 64, "H": 64, "KVH": 8, "hd": 128, "page": 64, "dtype": "bf16", "prefix": 16384, "max_suffix": 1024, "lens": 10},
        # one sequence's logits: penalties alone
        {"name": "logits_1", "op": "logits", "B": 1, "V": V_LLAMA, "hist": 768, "xtype": "f32", "bias": 0, "masks": 0, "lens": 11},
        # a serving batch's logits: long histories, some requests under a grammar, some with biases
        {"name": "logits_64", "op": "logits", "B": 64, "V": V_LLAMA, "hist": 8192, "xtype": "f32", "bias": 300, "masks": 24, "lens": 12},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attn", "attn", "attn", "prefix", "prefix", "logits"])
    lens = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64, 128, 256])
    hd = rng.choice([64, 128, 128])
    KVH = rng.choice([1, 2, 4, 8])
    H = KVH * rng.choice([1, 2, 3, 4, 7, 8, 16])
    dtype = rng.choice(["f16", "bf16"])
    if op == "plan":
        fresh = rng.choice([1, _log(rng, 2, 1024)])
        return {"op": op, "B": _log(rng, 1, 1024), "page": page, "max_cached": _log(rng, 1, 8192), "max_fresh": fresh, "tight": rng.random() < 0.5, "lens": lens}
    if op == "append":
        return {"op": op, "T": _log(rng, 1, 16384), "KVH": KVH, "hd": hd, "page": page, "xtype": rng.choice(["f32", "f16", "bf16"]), "dtype": dtype, "lens": lens}
    if op == "attn":
        rows = rng.choice([1, 1, _log(rng, 2, 4096)])
        n = _log(rng, max(16, rows), 32768 if rows == 1 else max(2 * rows, 8192))
        # no more than the largest listed ones: cached values for single rows, scores for many
        most = 64 * 32768 * 8 * 128 // (n * KVH * hd) if rows == 1 else 32 * 8192 * 8192 // (rows * n * H)
        B = _log(rng, 1, max(1, min(64, most)))
        window = rng.choice([None, _log(rng, 1, 2 * n)])
        return {"op": op, "B": B, "H": H, "KVH": KVH, "hd": hd, "page": page, "dtype": dtype, "max_rows": rows, "max_len": n,
                "window": window, "sinks": 0 if window is None else rng.choice([0, _log(rng, 1, 64)]), "lens": lens}
    if op == "prefix":
        return {"op": op, "B": _log(rng, 1, 64), "H": H, "KVH": KVH, "hd": hd, "page": page, "dtype": dtype, "prefix": _log(rng, 1, 16384),
                "max_suffix": _log(rng, 1, 1024), "lens": lens}
    return {"op": op, "B": _log(rng, 1, 64), "V": rng.choice([V_LLAMA, _log(rng, 256, 152064)]), "hist": _log(rng, 1, 8192),
            "xtype": rng.choice(["f32", "f16", "bf16"]), "bias": rng.choice([0, _log(rng, 1, 300)]), "masks": rng.choice([0, _log(rng, 1, 64)]), "lens": lens}


def _shape(c):
    """The lengths of a case, by the case alone: the work does not depend on the seed."""
    r = random.Random(c["lens"])
    B = c.get("B", 0)
    if c["op"] == "plan":
        cached = [_log(r, 1, c["max_cached"]) - 1 for _ in range(B)]
        fresh = [1 if c["max_fresh"] == 1 else _log(r, 1, c["max_fresh"]) for _ in range(B)]
        for b in range(B):
            if r.random() < 0.05:  # an idle slot
                fresh[b] = 0
        return {"cached": cached, "fresh": fresh}
    if c["op"] == "append":
        return {"dropped": [r.random() < 0.03 for _ in range(c["T"])]}
    if c["op"] == "attn":
        n, m = c["max_len"], c["max_rows"]
        lens = [n] + [r.randint(max(1, n // 8), n) for _ in range(B - 1)]
        if B >= 6:
            lens[B // 2] = 0  # an idle slot: its rows see nothing
        rows = [1 if m == 1 else min(x, _log(r, 1, m)) for x in lens]
        rows[0] = m
        return {"lens": lens, "rows": rows}
    if c["op"] == "prefix":
        return {"lens": [c["prefix"] + r.randint(1, c["max_suffix"]) for _ in range(B)]}
    total = [c["hist"]] + [r.randint(0, c["hist"]) for _ in range(B - 1)]
    return {"total": total, "prompt": [r.randint(0, t) for t in total], "mask_row": [r.randrange(-1, c["masks"]) if c["masks"] else -1 for _ in range(B)],
            "nbias": [r.randint(0, c["bias"]) for _ in range(B)]}


def _ceil(a, b):
    return -(-a // b)


def _plan_counts(c, sh):
    """(pages each request lacks, which requests get theirs, free pages, rows)"""
    need = [_ceil(a + f, c["page"]) - _ceil(a, c["page"]) for a, f in zip(sh["cached"], sh["fresh"])]
    free = int(0.9 * sum(need)) if c["tight"] else sum(need) + 7
    ok, run = [], 0
    for n in need:
        run += n
        ok.append(n == 0 or run <= free)
    return need, ok, free, sum(sh["fresh"])


def work(case):
    c, sh = case, _shape(case)
    if c["op"] == "plan":
        need, ok, _, T = _plan_counts(c, sh)
        new = sum(n for n, o in zip(need, ok) if o)
        # lengths in, offsets and lengths out, a page number read and written per new page, one read per request, slot and position per row
        return {"bytes": c["B"] * (8 + 8 + 4) + 8 * new + 12 * (T + 5), "flops": 0}
    if c["op"] == "append":
        n = c["T"] - sum(sh["dropped"])
        return {"bytes": 2 * n * c["KVH"] * c["hd"] * (SIZE[c["xtype"]] + SIZE[c["dtype"]]) + 8 * c["T"], "flops": 0}
    if c["op"] == "attn":
        kv = pairs = 0
        for n, m in zip(sh["lens"], sh["rows"]):
            seen = 0
            for i in range(m):
                p = n - m + i
                if p < 0:
                    continue
                w = p + 1 if c["window"] is None else min(c["window"], p + 1)
                seen += w + min(c["sinks"], p + 1 - w)
            pairs += seen
            lo = 0 if c["window"] is None else max(0, n - m - c["window"] + 1)  # the first row's window on
            kv += (n - lo) + min(c["sinks"], lo) if n else 0
        T = sum(sh["rows"])
        return {"bytes": 2 * kv * c["KVH"] * c["hd"] * 2 + 2 * T * c["H"] * c["hd"] * 2, "flops": 4 * pairs * c["H"] * c["hd"]}
    if c["op"] == "prefix":
        kv = c["prefix"] + sum(n - c["prefix"] for n in sh["lens"])
        return {"bytes": 2 * kv * c["KVH"] * c["hd"] * 2 + 2 * c["B"] * c["H"] * c["hd"] * 2, "flops": 4 * sum(sh["lens"]) * c["H"] * c["hd"]}
    words = _ceil(c["V"], 32)
    return {"bytes": c["B"] * c["V"] * (SIZE[c["xtype"]] + 4) + 8 * sum(sh["total"]) + 8 * sum(sh["nbias"]) + 4 * words * len({m for m in sh["mask_row"] if m >= 0}),
            "flops": 0}


# ---------------------------------------------------------------- the inputs

def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _pools(c, n_pages, g):
    """K and V pools [pages, KV heads, positions of a page, head dim]"""
    shape = (n_pages, c["KVH"], c["page"], c["hd"])
    k = torch.randn(shape, generator=g, device="cuda", dtype=DT[c["dtype"]])
    v = torch.randn(shape, generator=g, device="cuda", dtype=DT[c["dtype"]])
    return k, v


def _tables(lens, page, first, spare, g):
    """Block tables of shuffled pages from `first` on (-1 past a request's own), and how many pages there are."""
    n = [_ceil(x, page) for x in lens]
    wide, total = max(1, max(n)), first + sum(n) + spare
    perm = (torch.randperm(total - first, generator=g, device="cuda") + first).to(torch.int32)
    t = torch.full((len(lens), wide), -1, dtype=torch.int32, device="cuda")
    live = torch.arange(wide, device="cuda")[None, :] < _i32(n)[:, None]
    t[live] = perm[: sum(n)]
    return t, perm[sum(n):], total


def prepare(case, seed):
    c, sh, g = case, _shape(case), _gen(seed)
    s = {"case": c}
    if own:
        s["ctx"] = _context()  # a handle, as a program keeps it
    if c["op"] == "plan":
        need, _, n_free, T = _plan_counts(c, sh)
        lens = sh["cached"]
        s["tables"], free, _ = _tables(lens + [a + f for a, f in zip(lens, sh["fresh"])], c["page"], 0, n_free + 3, g)
        s["tables"] = s["tables"][: c["B"]].contiguous()  # as wide as the longest request gets
        s["free"] = free.contiguous()
        s["n_free"] = _i32([n_free])
        s["cached"], s["fresh"] = _i32(lens), _i32(sh["fresh"])
        cap = T + 5  # a padded batch
        s["row_start"], s["kv_len"] = _i32([0] * (c["B"] + 1)), _i32([0] * c["B"])
        s["slots"] = torch.zeros(cap, dtype=torch.int64, device="cuda")
        s["positions"], s["left"] = _i32([0] * cap), _i32([0])
        return s
    if c["op"] == "append":
        T = c["T"]
        n_pages = _ceil(T, c["page"]) + 3
        k, v = _pools(c, n_pages + 1, g)
        s["k_all"], s["v_all"] = k, v  # one page more: where the plain form puts dropped rows
        x = torch.randn((T, (2 * c["KVH"] + 3) * c["hd"]), generator=g, device="cuda", dtype=torch.float32).to(DT[c["xtype"]])
        n = c["KVH"] * c["hd"]
        s["k"], s["v"] = x[:, 3 * c["hd"]: 3 * c["hd"] + n], x[:, 3 * c["hd"] + n:]  # parts of the projection's rows
        slots = torch.randperm(n_pages * c["page"], generator=g, device="cuda")[:T]
        s["slots"] = torch.where(torch.tensor(sh["dropped"], device="cuda"), torch.full_like(slots, -1), slots)
        if own:
            from tcb_b200 import serve

            s["pages"] = serve.Pages(s["ctx"], k[:n_pages], v[:n_pages])
        return s
    if c["op"] == "attn":
        lens, rows = sh["lens"], sh["rows"]
        s["tables"], _, total = _tables(lens, c["page"], 0, 2, g)
        s["k"], s["v"] = _pools(c, total, g)
        T, start = sum(rows), [0]
        for m in rows:
            start.append(start[-1] + m)
        s["q"] = (2.0 * torch.randn((T, c["H"], c["hd"]), generator=g, device="cuda")).to(DT[c["dtype"]])
        s["out"] = torch.empty_like(s["q"])
        s["row_start"], s["kv_len"] = _i32(start), _i32(lens)
        if own:
            from tcb_b200 import serve

            s["pages"] = serve.Pages(s["ctx"], s["k"], s["v"])
        return s
    if c["op"] == "prefix":
        lens, P = sh["lens"], c["prefix"]
        whole = P // c["page"]  # pages that hold nothing but the prefix
        own_lens = [n - whole * c["page"] for n in lens]
        first = _ceil(P, c["page"])
        t, _, total = _tables(own_lens, c["page"], first, 2, g)
        s["tables"] = torch.cat([torch.full((c["B"], whole), -1, dtype=torch.int32, device="cuda"), t], 1).contiguous()
        s["prefix"] = torch.randperm(first, generator=g, device="cuda").to(torch.int32)
        s["k"], s["v"] = _pools(c, total, g)
        s["q"] = (2.0 * torch.randn((c["B"], c["H"], c["hd"]), generator=g, device="cuda")).to(DT[c["dtype"]])
        s["out"] = torch.empty_like(s["q"])
        s["kv_len"] = _i32(lens)
        if own:
            from tcb_b200 import serve

            s["pages"] = serve.Pages(s["ctx"], s["k"], s["v"])
        return s
    B, V = c["B"], c["V"]
    s["logits"] = (3.0 * torch.randn((B, V), generator=g, device="cuda")).to(DT[c["xtype"]])
    s["out"] = torch.empty((B, V), dtype=torch.float32, device="cuda")
    s["token"] = torch.empty(B, dtype=torch.int64, device="cuda")
    # token ids as text has them: few are frequent
    s["history"] = (V * torch.rand((B, c["hist"]), generator=g, device="cuda") ** 3).to(torch.int64).clamp_(max=V - 1)
    s["total"], s["prompt"] = _i32(sh["total"]), _i32(sh["prompt"])
    s["repetition"] = 1.0 + 0.5 * torch.rand(B, generator=g, device="cuda")
    s["frequency"] = 0.5 * torch.rand(B, generator=g, device="cuda")
    s["presence"] = 0.5 * torch.rand(B, generator=g, device="cuda")
    s["bias_ids"] = s["bias"] = s["mask"] = s["mask_row"] = None
    if c["bias"]:
        # distinct ids in a row, -1 past a request's own
        ids = torch.rand((B, V), generator=g, device="cuda").topk(min(c["bias"], V), dim=1).indices.to(torch.int32)
        s["bias_ids"] = torch.where(torch.arange(ids.shape[1], device="cuda")[None] < _i32(sh["nbias"])[:, None], ids, torch.full_like(ids, -1))
        s["bias"] = 2.0 * torch.randn(ids.shape, generator=g, device="cuda")
    if c["masks"]:
        # from a few allowed tokens to nearly all
        share = torch.rand((c["masks"], 1), generator=g, device="cuda") ** 2
        bit = torch.rand((c["masks"], _ceil(V, 32) * 32), generator=g, device="cuda") < share
        words = (bit.view(c["masks"], -1, 32).to(torch.int64) << torch.arange(32, device="cuda")).sum(2)
        s["mask"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
        s["mask_row"] = _i32(sh["mask_row"])
    return s


# ---------------------------------------------------------------- the passes

def run(s):
    c = s["case"]
    return globals()["_run_" + c["op"] if own else "_plain_" + c["op"]](s, c)


def _run_plan(s, c):
    from tcb_b200 import serve

    serve.plan(s["ctx"], c["page"], s["cached"], s["fresh"], s["tables"], s["free"], s["n_free"], s["row_start"], s["kv_len"], s["slots"], s["positions"], s["left"])
    return {k: s[k] for k in ("tables", "row_start", "kv_len", "slots", "positions", "left")}


def _run_append(s, c):
    s["pages"].append(s["k"], s["v"], s["slots"])
    return {"k": s["k_all"][:-1], "v": s["v_all"][:-1]}


def _run_attn(s, c):
    s["pages"].attend(s["q"], s["out"], s["row_start"], s["kv_len"], s["tables"], c["max_rows"], c["max_len"], window=c["window"], sinks=c["sinks"])
    return s["out"]


def _run_prefix(s, c):
    s["pages"].attend_prefix(s["q"], s["out"], s["prefix"], c["prefix"], s["kv_len"], s["tables"], c["prefix"] + c["max_suffix"])
    return s["out"]


def _run_logits(s, c):
    from tcb_b200 import serve

    serve.penalize(s["ctx"], s["logits"], s["out"], s["token"], history=s["history"], prompt_len=s["prompt"], total_len=s["total"], repetition=s["repetition"],
                   frequency=s["frequency"], presence=s["presence"], bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"], mask_row=s["mask_row"])
    return {"logits": s["out"], "token": s["token"]}


def _plain_plan(s, c):
    page, tables, free = c["page"], s["tables"], s["free"]
    cap, wide = s["slots"].numel(), tables.shape[1]
    cached, fresh, n_free = s["cached"].long(), s["fresh"].long(), s["n_free"].long()
    end = torch.cumsum(fresh, 0)
    row_start = torch.cat([torch.zeros_like(end[:1]), end]).clamp(max=cap)
    fits = (end <= cap) & (cached + fresh <= wide * page)
    have = (cached + page - 1) // page
    need = torch.where(fits, (cached + fresh + page - 1) // page - have, torch.zeros_like(have))
    last = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (last <= n_free))
    j = torch.arange(wide, device="cuda")[None, :] - have[:, None]
    new = granted[:, None] & (j >= 0) & (j < need[:, None])
    at = (n_free - 1 - (last - need)[:, None] - j).clamp(0, free.numel() - 1)
    tables = torch.where(new, free[at], tables)
    left = n_free - torch.where(granted, last, torch.zeros_like(last)).max()
    r = torch.arange(cap, device="cuda")
    b = torch.searchsorted(row_start[1:].contiguous(), r, right=True).clamp(max=c["B"] - 1)
    pos = cached[b] + r - row_start[b]
    ok = granted[b] & (r < row_start[-1])
    at = torch.where(ok, pos, torch.zeros_like(pos))
    slots = torch.where(ok, tables[b, at // page].long() * page + at % page, torch.full_like(pos, -1))
    return {"tables": tables, "row_start": row_start.int(), "kv_len": torch.where(granted, cached + fresh, torch.zeros_like(cached)).int(), "slots": slots,
            "positions": torch.where(ok, pos, torch.full_like(pos, -1)).int(), "left": left.int()}


def _plain_append(s, c):
    page, n = c["page"], s["k_all"].shape[0] - 1
    slot = torch.where(s["slots"] < 0, torch.full_like(s["slots"], n * page), s["slots"])  # dropped rows: the page past the pool
    s["k_all"].permute(0, 2, 1, 3)[slot // page, slot % page] = s["k"].float().view(-1, c["KVH"], c["hd"]).to(DT[c["dtype"]])
    s["v_all"].permute(0, 2, 1, 3)[slot // page, slot % page] = s["v"].float().view(-1, c["KVH"], c["hd"]).to(DT[c["dtype"]])
    return {"k": s["k_all"][:-1], "v": s["v_all"][:-1]}


def _gather(pool, tables, n):
    """[B, KVH, n, hd] in 32 bits: the first n positions that a table names"""
    B, (_, KVH, page, hd) = tables.shape[0], pool.shape
    return pool[tables.clamp(min=0).long()].float().permute(0, 2, 1, 3, 4).reshape(B, KVH, -1, hd)[:, :, :n]


def _softmax(x, visible):
    """softmax over the visible scores; a row that sees nothing gives zeros"""
    x = torch.where(visible, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_attn(s, c):
    B, H, KVH, hd, m = c["B"], c["H"], c["KVH"], c["hd"], c["max_rows"]
    start, n = s["row_start"].long(), s["kv_len"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(m, device="cuda")
    at = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)  # a request's rows side by side, padded
    q = s["q"].float()[at].view(B, m, KVH, H // KVH, hd).permute(0, 2, 3, 1, 4).reshape(B, KVH, -1, hd)
    k, v = _gather(s["k"], s["tables"], c["max_len"]), _gather(s["v"], s["tables"], c["max_len"])
    j = torch.arange(k.shape[2], device="cuda")
    v = torch.where((j < n[:, None])[:, None, :, None], v, torch.zeros_like(v))
    pos = (n - count)[:, None] + i
    sees = j <= pos[:, :, None]
    if c["window"] is not None:
        sees = sees & ((j > pos[:, :, None] - c["window"]) | (j < c["sinks"]))
    sees = sees & (j < n[:, None, None])
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    p = _softmax(x.view(B, KVH, H // KVH, m, -1), sees[:, None, None]).view_as(x)
    o = torch.matmul(p, v).view(B, KVH, H // KVH, m, hd).permute(0, 3, 1, 2, 4).reshape(B * m, H, hd)
    r = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(start[1:].contiguous(), r, right=True)
    return o[b * m + r - start[b]].to(DT[c["dtype"]])


def _plain_prefix(s, c):
    B, H, KVH, hd, P, page = c["B"], c["H"], c["KVH"], c["hd"], c["prefix"], c["page"]
    n = s["kv_len"].long()
    skip = P // page
    q = s["q"].float().view(B, KVH, H // KVH, hd)
    kp, vp = _gather(s["k"], s["prefix"][None], P)[0], _gather(s["v"], s["prefix"][None], P)[0]
    ks, vs = (_gather(s[x], s["tables"][:, skip:], c["max_suffix"] + page) for x in ("k", "v"))
    j = skip * page + torch.arange(ks.shape[2], device="cuda")
    sees = (j >= P) & (j < n[:, None])
    vs = torch.where(sees[:, None, :, None], vs, torch.zeros_like(vs))
    x = torch.cat([torch.matmul(q.permute(1, 0, 2, 3).reshape(KVH, -1, hd), kp.transpose(1, 2)).view(KVH, B, H // KVH, P).permute(1, 0, 2, 3),
                   torch.matmul(q, ks.transpose(2, 3))], -1) * (1.0 / math.sqrt(hd))
    sees = torch.cat([torch.arange(P, device="cuda") < n[:, None], sees], 1)
    p = _softmax(x, sees[:, None, None])
    o = torch.matmul(p[..., :P].permute(1, 0, 2, 3).reshape(KVH, -1, P), vp).view(KVH, B, H // KVH, hd).permute(1, 0, 2, 3) + torch.matmul(p[..., P:], vs)
    return o.reshape(B, H, hd).to(DT[c["dtype"]])


def _plain_logits(s, c):
    B, V = c["B"], c["V"]
    x = s["logits"].float()
    at = torch.arange(s["history"].shape[1], device="cuda")[None]
    made = ((at >= s["prompt"][:, None]) & (at < s["total"][:, None])).int()
    live = (at < s["total"][:, None]).int()
    n = torch.zeros((B, V), dtype=torch.int32, device="cuda").scatter_add_(1, s["history"], made)
    seen = torch.zeros((B, V), dtype=torch.int32, device="cuda").scatter_add_(1, s["history"], live) > 0
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * n.float()
    x = torch.where(n > 0, x - s["presence"][:, None], x)
    if s["bias"] is not None:
        add = torch.zeros((B, V + 1), dtype=torch.float32, device="cuda")  # the last column takes the unused entries
        add.scatter_(1, torch.where(s["bias_ids"] < 0, torch.full_like(s["bias_ids"], V), s["bias_ids"]).long(), s["bias"])
        x = x + add[:, :V]
    if s["mask"] is not None:
        v = torch.arange(V, device="cuda")
        bit = (s["mask"][:, v // 32] >> (v % 32)) & 1
        free = s["mask_row"] < 0
        ok = (bit[s["mask_row"].clamp(min=0).long()] != 0) | free[:, None]
        x = torch.where(ok, x, torch.full_like(x, -math.inf))
    top = x.amax(1, keepdim=True)
    ids = torch.arange(V, device="cuda").expand(B, V)
    first = torch.where(x == top, ids, torch.full_like(ids, V)).amin(1)
    return {"logits": x, "token": torch.where(torch.isinf(top[:, 0]), torch.full_like(first, -1), first)}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None  # whole numbers
    s, sh = prepare(case, seed), _shape(case)
    if c["op"] == "append":
        out = {}
        for name in ("k", "v"):
            pool = s[name + "_all"][:-1].double()
            rows = s[name].double().view(c["T"], c["KVH"], c["hd"])
            keep = s["slots"] >= 0
            pool.transpose(1, 2)[s["slots"][keep] // c["page"], s["slots"][keep] % c["page"]] = rows[keep]
            out[name] = pool
        return out
    if c["op"] in ("attn", "prefix"):
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        G, r0 = c["H"] // c["KVH"], 0
        for b, n in enumerate(sh["lens"]):
            m = sh["rows"][b] if c["op"] == "attn" else 1
            at = torch.arange(n, device="cuda")
            page = s["tables"][b][at // c["page"]].long()
            if c["op"] == "prefix":
                first = torch.arange(c["prefix"], device="cuda")
                page[: c["prefix"]] = s["prefix"][first // c["page"]].long()
            p = torch.arange(n - m, n, device="cuda")[:, None]
            sees = at[None] <= p
            if c.get("window") is not None:
                sees &= (at[None] > p - c["window"]) | (at[None] < c["sinks"])
            for h in range(c["KVH"] if n else 0):
                k, v = (s[x][page, h, at % c["page"]].double() for x in ("k", "v"))
                for q in range(h * G, h * G + G):
                    x = s["q"][r0:r0 + m, q].double() @ k.T / math.sqrt(c["hd"])
                    x = x.masked_fill(~sees, -math.inf)
                    out[r0:r0 + m, q] = torch.softmax(x, 1) @ v
            r0 += m
        return out
    x = s["logits"].double()
    for b, (total, prompt) in enumerate(zip(sh["total"], sh["prompt"])):
        seen = torch.bincount(s["history"][b, :total], minlength=c["V"])
        n = torch.bincount(s["history"][b, prompt:total], minlength=c["V"])
        r = s["repetition"][b].double()
        hit = seen > 0
        x[b, hit] = torch.maximum(x[b, hit], torch.zeros_like(x[b, hit])) / r + torch.minimum(x[b, hit], torch.zeros_like(x[b, hit])) * r
        x[b] -= s["frequency"][b].double() * n + s["presence"][b].double() * (n > 0)
        if c["bias"]:
            k = sh["nbias"][b]
            x[b, s["bias_ids"][b, :k].long()] += s["bias"][b, :k].double()
        if sh["mask_row"][b] >= 0:
            words = s["mask"][sh["mask_row"][b]].long()
            bits = ((words[:, None] >> torch.arange(32, device="cuda")) & 1).view(-1)[: c["V"]]
            x[b, bits == 0] = -math.inf
    return {"logits": x, "token": None}
