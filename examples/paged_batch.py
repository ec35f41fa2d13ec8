"""Greedy decoding of a batch of requests over a paged K/V cache: the serving
operators (tcb_b200.serve) run together around the quantized products, on a
small Llama-shaped model with random weights.

    python examples/paged_batch.py

Every step plans the pages of its new positions (serve.plan), and per layer
appends the K/V rows (Pages.append) and attends (Pages.attend, or
Pages.attend_prefix for a decode step behind a shared first text); the last
step of all is the pick (serve.penalize).  RMSNorm, rotary embedding and SwiGLU
are plain torch operations here; the decoder engine (tcb_b200.llama) has them
fused, over a cache of its own for each sequence.
"""
from __future__ import annotations

import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import tcb_b200 as T  # noqa: E402
from tcb_b200 import llama, serve  # noqa: E402


class PagedBatch:
    """One batch of requests over `n_pages` pages of `page` positions a layer."""

    def __init__(self, ctx, model: dict, batch: int, n_pages: int, page: int = 16, window=None, sinks: int = 0):
        c = model["cfg"]
        self.ctx, self.m, self.c, self.page, self.window, self.sinks = ctx, model, c, page, window, sinks
        shape = (n_pages, c.n_kv_heads, page, c.head_dim)
        self.layers = [serve.Pages(ctx, *(torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in "kv"))
                       for _ in range(c.n_layers)]
        i32 = dict(dtype=torch.int32, device="cuda")
        self.free = torch.randperm(n_pages, device="cuda").to(torch.int32)
        self.n_free = torch.full((1,), n_pages, **i32)
        self.tables = torch.full((batch, -(-c.max_ctx // page)), -1, **i32)
        self.cached = torch.zeros(batch, **i32)
        self.row_start, self.kv_len = torch.empty(batch + 1, **i32), torch.empty(batch, **i32)
        self.balance, self.taken = torch.empty(1, **i32), torch.empty(1, **i32)
        self.prefix, self.prefix_len = None, 0
        f = torch.tensor([c.rope_theta ** (-2.0 * i / c.head_dim) for i in range(c.head_dim // 2)], dtype=torch.float32)
        ang = (torch.arange(c.max_ctx, dtype=torch.float32)[:, None] * f).double()
        self.cos, self.sin = ang.cos().float().cuda(), ang.sin().float().cuda()

    def _product(self, kind: str, w, x, rows: int):
        out = torch.empty((x.shape[0], rows), dtype=torch.float32, device="cuda")
        return self.ctx.qgemm(llama.TYPES[kind], w, x.contiguous(), out)

    def _rms(self, x, w):
        return x / torch.sqrt(x.square().mean(1, keepdim=True) + self.c.eps) * w

    def step(self, rows: list) -> torch.Tensor:
        """Feed rows[b] (token ids) to request b; the logits of every request's
        last row, float32 [batch, vocab] (an idle request's row is its last
        one's again)."""
        c, sh = self.c, llama.shapes(self.c)
        H, KVH, hd = c.n_heads, c.n_kv_heads, c.head_dim
        fresh = torch.tensor([len(r) for r in rows], dtype=torch.int32, device="cuda")
        ids = np.concatenate([np.asarray(r, np.int64) for r in rows])
        n, most = len(ids), max(len(r) for r in rows)
        slots = torch.empty(n, dtype=torch.int64, device="cuda")
        pos = torch.empty(n, dtype=torch.int32, device="cuda")
        serve.plan(self.ctx, self.page, self.cached, fresh, self.tables, self.free, self.n_free, self.row_start,
                   self.kv_len, slots, pos, self.balance, self.taken)
        if self.balance.item() < 0 or (self.kv_len < fresh).any():
            raise RuntimeError("the pages do not hold the batch")
        self.n_free -= self.taken
        self.cached.copy_(self.kv_len)
        single = most == 1 and n == len(rows)
        x = torch.empty((n, c.d_model), dtype=torch.float32, device="cuda")
        self.ctx.qembed(llama.TYPES["tok_emb"], self.m["tok_emb"], c.vocab, c.d_model, ids, x)
        cos, sin = self.cos[pos.long(), None], self.sin[pos.long(), None]
        for l, pages in enumerate(self.layers):
            qkv = self._product("qkv", self.m["qkv"][l], self._rms(x, self.m["attn_norm"][l]), sh["qkv"][0])
            a, b = qkv[:, :(H + KVH) * hd].view(n, H + KVH, 2, hd // 2).unbind(2)
            rot = torch.cat([a * cos - b * sin, a * sin + b * cos], 2).view(n, (H + KVH) * hd)
            pages.append(rot[:, H * hd:], qkv[:, (H + KVH) * hd:], slots)
            q = rot[:, :H * hd].half().view(n, H, hd)
            att = torch.zeros_like(q)
            if single and self.prefix is not None and self.window is None:
                pages.attend_prefix(q, att, self.prefix, self.prefix_len, self.kv_len, self.tables, c.max_ctx)
            else:
                pages.attend(q, att, self.row_start, self.kv_len, self.tables, most, c.max_ctx, window=self.window,
                             sinks=self.sinks)
            x = x + self._product("o", self.m["o"][l], att.float().view(n, H * hd), c.d_model)
            gu = self._product("gate_up", self.m["gate_up"][l], self._rms(x, self.m["ffn_norm"][l]), sh["gate_up"][0])
            g, u = gu.chunk(2, 1)
            x = x + self._product("down", self.m["down"][l], torch.nn.functional.silu(g) * u, c.d_model)
        last = x[(self.row_start[1:].long() - 1).clamp(min=0)]
        return self._product("head", self.m["head"], self._rms(last, self.m["final_norm"]), c.vocab)

    def share(self, tokens):
        """Feed `tokens` once and make them the first text of every request
        (before any other step; their whole pages are shared, so their number is
        held to a multiple of the page): the tokens shared."""
        n = len(tokens) // self.page * self.page
        if n == 0:
            return 0
        self.step([tokens[:n]] + [[] for _ in range(len(self.cached) - 1)])
        self.prefix_len, self.prefix = n, self.tables[0, :n // self.page].clone()
        self.tables[:, :n // self.page] = self.prefix
        self.cached.fill_(n)
        return n


def generate(batch: PagedBatch, prompts: list, steps: int, shared: int = 0, chunk: int = 12, **penalties):
    """Prompts (lists of token ids, the first `shared` of them equal) and then
    `steps` greedy tokens of every request.  A prompt is fed at most `chunk`
    tokens a step, so that a long one does not hold up the others' tokens:
    (token history int64 [batch, width], lengths, and for every request the logits
    that its tokens were picked from)."""
    B, width = len(prompts), max(len(p) for p in prompts) + steps
    history = torch.full((B, width), -1, dtype=torch.int64, device="cuda")
    for b, p in enumerate(prompts):
        history[b, :len(p)] = torch.as_tensor(p, device="cuda")
    prompt_len = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
    total = prompt_len.clone()
    done = batch.share(prompts[0][:shared]) if shared else 0
    pending, seen = [list(p[done:]) for p in prompts], [[] for _ in prompts]
    token = torch.empty(B, dtype=torch.int64, device="cuda")
    while min(len(s) for s in seen) < steps:
        rows = [p[:chunk] for p in pending]
        pending = [p[chunk:] for p in pending]
        logits = batch.step(rows)
        serve.penalize(batch.ctx, logits, torch.empty_like(logits), token, history=history, prompt_len=prompt_len,
                       total_len=total, **penalties)
        for b, t in enumerate(token.tolist()):
            if rows[b] and not pending[b] and len(seen[b]) < steps:  # the request's last row: its next token
                seen[b].append(logits[b])
                history[b, len(prompts[b]) + len(seen[b]) - 1] = t
                total[b] += 1
                pending[b] = [t] if len(seen[b]) < steps else []
    return history, total, seen


def main():
    cfg = llama.LlamaConfig(n_layers=2, d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, ffn_dim=1024, vocab=2048,
                            max_ctx=160)
    ctx = T.Context(0)
    model = llama.device_model(cfg, 15, llama.host_model(cfg, seed=15, varied=True))
    first = [17, 901, 5, 1333, 42, 2047, 0, 777] * 3
    prompts = [first + [3, 99], first + [7], first + [500, 501, 502, 503], first + [1]]
    for name, kw in (("greedy", {}), ("repetition 1.3", {"repetition": torch.full((4,), 1.3, device="cuda")})):
        history, total, _ = generate(PagedBatch(ctx, model, 4, 64), prompts, 24, shared=len(first), **kw)
        print(name)
        for h, n, p in zip(history.tolist(), total.tolist(), prompts):
            print("  ", h[len(p):n])


if __name__ == "__main__":
    main()
