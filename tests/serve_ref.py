"""Plain 64-bit restatements of the serving operators (include/tcb.h), one
request at a time, and the bounds their 16-bit results are held to."""
import math

import torch


def plan(page, cached, fresh, tables, free, n_free, rows):
    """tcb_page_plan on Python lists (tables and free are copied)."""
    tables, width = [list(t) for t in tables], len(tables[0]) if tables else 0
    n = max(0, min(n_free, len(free)))
    row, asked, taken, last = 0, 0, 0, 0
    row_start, kv_len, slots, positions = [], [], [-1] * rows, [-1] * rows
    for b, (c, f) in enumerate(zip(cached, fresh)):
        r0 = row
        row_start.append(min(row, rows))
        row += max(f, 0)
        fits = c >= 0 and f >= 0 and row <= rows and c + f <= width * page
        have = -(-c // page)
        need = -(-(c + f) // page) - have if fits else 0
        ok = fits and (need == 0 or asked + need <= n)
        if ok:
            for j in range(need):
                tables[b][have + j] = free[n - 1 - asked - j]
            if need:
                taken = asked + need
            last = asked + need
            for i in range(f):
                p = c + i
                positions[r0 + i] = p
                g = tables[b][p // page]
                slots[r0 + i] = g * page + p % page if g >= 0 else -1
        kv_len.append(c + f if ok else 0)
        asked += need
    return tables, row_start + [min(row, rows)], kv_len, slots, positions, n - last, taken


def attention(q, k, v, pos, scale, window=None, sinks=0):
    """q [n, H, hd], k and v [len, KVH, hd] in float64, pos the rows'
    positions: (out, sum of p |v|) of every row, zeros where nothing is
    visible.  Keys that a row does not see are left out, not multiplied by 0."""
    n, H, hd = q.shape
    G = H // k.shape[1]
    out = torch.zeros(n, H, hd, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i in range(n):
        p = pos[i]
        js = [j for j in range(p + 1) if window is None or j > p - window or j < sinks]
        if not js:
            continue
        js = torch.tensor(js, device=q.device)
        s = torch.einsum("kgd,jkd->kgj", q[i].view(-1, G, hd), k[js]) * scale
        w = torch.softmax(s, -1)
        out[i] = torch.einsum("kgj,jkd->kgd", w, v[js]).reshape(H, hd)
        mag[i] = torch.einsum("kgj,jkd->kgd", w, v[js].abs()).reshape(H, hd)
    return out, mag


def attention_bound(out, mag, n_keys, dtype):
    """Per element: the weights are rounded to the cache's type before the
    product with v (relative u, or half the least subnormal of f16, on
    weights whose largest is at least 1 times a power of two above it), the
    sum they are divided by may be of the unrounded ones (another u of the
    result), and the result is rounded once; the f32 scores, exponentials and
    sums add a few parts in 10^6."""
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    vmax = mag.abs().max() if mag.numel() else 0.0
    return u * mag * (1 + u) + 2 * u * out.abs() + 2e-5 * mag + tiny * (1 + 4 * n_keys * vmax)


def penalties(x, history, prompt, total, rep, freq, pres, bias, allowed):
    """One row of logits in float64.  bias: list of (token, value); allowed:
    bool tensor or None."""
    V = x.shape[0]
    x = x.clone()
    seen, made = {}, {}
    for i, t in enumerate(history[:total]):
        if 0 <= t < V:
            seen[t] = True
            if i >= prompt:
                made[t] = made.get(t, 0) + 1
    for t in seen:
        x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
    for t, n in made.items():
        x[t] = x[t] - freq * n - pres
    for t, b in {t: b for t, b in bias if 0 <= t < V}.items():
        x[t] = x[t] + b
    if allowed is not None:
        x[~allowed] = -math.inf
    return x
