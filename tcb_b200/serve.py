"""Serving operators over a paged K/V cache (include/tcb.h, tcb_page_* and
tcb_logits_penalize): a thin ctypes view for torch CUDA tensors.

One step of a batch of requests:
  plan(...)             pages, row offsets, slots and positions of the step
  Pages.append(...)     the step's K/V rows into the cache
  Pages.attend(...)     causal attention over the pages, with a sliding
                        window and first positions that stay visible
  Pages.attend_prefix(...)  a decode step of a batch over one shared prefix
  penalize(...)         penalties, biases and masks on the logits, the pick
All lengths and page numbers are int32 tensors on the device; nothing here
waits for the device.  Every call runs on `stream` (the current one when it is
None), and calls on one context are to be ordered on one stream.  Device-side
findings (a page outside the pool, a length past max_len) are read with
Context.device_error().
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import BF16, F16, F32, TcbError, lib

_TYPE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_I32, _I64 = torch.int32, torch.int64


class _KvPages(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("dtype", ctypes.c_int), ("n_pages", ctypes.c_int),
                ("page", ctypes.c_int), ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("page_stride", ctypes.c_long), ("head_stride", ctypes.c_long), ("pos_stride", ctypes.c_long)]


class _LogitsArgs(ctypes.Structure):
    _fields_ = [("B", ctypes.c_int), ("V", ctypes.c_int),
                ("logits", ctypes.c_void_p), ("dtype", ctypes.c_int), ("ld", ctypes.c_long),
                ("out", ctypes.c_void_p), ("odtype", ctypes.c_int), ("ldo", ctypes.c_long),
                ("token", ctypes.c_void_p),
                ("history", ctypes.c_void_p), ("hist_width", ctypes.c_int), ("ldh", ctypes.c_long),
                ("prompt_len", ctypes.c_void_p), ("total_len", ctypes.c_void_p),
                ("repetition", ctypes.c_void_p), ("frequency", ctypes.c_void_p), ("presence", ctypes.c_void_p),
                ("bias_ids", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("n_bias", ctypes.c_int), ("ldb", ctypes.c_long),
                ("mask", ctypes.c_void_p), ("n_masks", ctypes.c_int), ("ldm", ctypes.c_long),
                ("mask_row", ctypes.c_void_p)]


def _stream(ctx, stream) -> int:
    """The handle of `stream`, or of the current stream of the context's device."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(ctx.device)
    return stream if isinstance(stream, int) else stream.cuda_stream


_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = lib()
        P, I, Lg, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
        L.tcb_page_plan.argtypes = [P, I, I, P, P, P, I, Lg, P, I, P, I, P, P, P, P, P, P, P]
        L.tcb_kv_append.argtypes = [P, P, I, P, Lg, P, Lg, I, P, P]
        L.tcb_page_attn.argtypes = [P, P, I, I, I, P, Lg, P, Lg, P, P, P, I, Lg, I, I, F, I, I, P]
        L.tcb_prefix_attn.argtypes = [P, P, I, I, P, Lg, P, Lg, P, I, P, P, I, Lg, I, F, P]
        L.tcb_logits_penalize.argtypes = [P, P, P]
        _bound = L
    return _bound


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _vec(t, n: int, dtype, name: str) -> int:
    """Address of a contiguous device vector of at least n elements."""
    if t.dtype is not dtype or not t.is_cuda or t.dim() != 1 or t.numel() < n or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} CUDA vector of at least {n} elements is wanted")
    return t.data_ptr()


def _rows(t, dtype, name: str):
    """(address, width, row stride) of a 2-D device tensor with dense rows."""
    if t.dtype is not dtype or not t.is_cuda or t.dim() != 2:
        raise ValueError(f"{name}: a 2-D {dtype} CUDA tensor with dense rows is wanted")
    (n, width), (ld, unit) = t.shape, t.stride()
    if width > 1 and unit != 1:
        raise ValueError(f"{name}: a 2-D {dtype} CUDA tensor with dense rows is wanted")
    return t.data_ptr(), width, ld if n > 1 else width


def plan(ctx, page, cached, fresh, tables, free, n_free, row_start, kv_len, slots, positions, balance, taken=None,
         stream=None):
    """tcb_page_plan: cached and fresh int32 [B]; tables int32 [B, width]
    (extended in place); free int32, the stack of free pages, of which the
    first n_free[0] are free; written: row_start int32 [B + 1], kv_len int32
    [B], slots int64 and positions int32 [rows], balance int32 [1] (the free
    pages left, below 0 the shortage), taken int32 [1] or None (pages taken)."""
    B, rows = cached.shape[0], slots.shape[0]
    tp, width, ldt = _rows(tables, _I32, "tables")
    _need(tables.shape[0] >= B, "tables: a row per request is wanted")
    rc = _lib().tcb_page_plan(ctx.handle, B, page, _vec(cached, B, _I32, "cached"), _vec(fresh, B, _I32, "fresh"), tp,
                              width, ldt, _vec(free, 0, _I32, "free"), free.shape[0], _vec(n_free, 1, _I32, "n_free"),
                              rows, _vec(row_start, B + 1, _I32, "row_start"), _vec(kv_len, B, _I32, "kv_len"),
                              _vec(slots, 0, _I64, "slots"), _vec(positions, rows, _I32, "positions"),
                              _vec(balance, 1, _I32, "balance"),
                              0 if taken is None else _vec(taken, 1, _I32, "taken"), _stream(ctx, stream))
    ctx._check(rc, "tcb_page_plan")


class Pages:
    """A paged K/V cache over two pools [pages, KV heads, positions of a
    page, head dim] (float16 or bfloat16 CUDA tensors of the same strides; a
    pool laid out otherwise is passed as its permuted view)."""

    def __init__(self, ctx, k, v):
        _need(k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride() and k.dtype == v.dtype,
              "k and v: two 4-D pools of one shape, type and strides are wanted")
        _need(k.is_cuda and v.is_cuda and k.device == v.device, "k and v: CUDA tensors of one device are wanted")
        _need(k.stride(3) == 1, "k and v: dense head elements are wanted")
        if k.dtype not in (torch.float16, torch.bfloat16):
            raise TcbError(2, "Pages")
        self.ctx, self.k, self.v = ctx, k, v
        n_pages, self.kv_heads, self.page, self.head_dim = k.shape
        self._kv = _KvPages(k.data_ptr(), v.data_ptr(), _TYPE[k.dtype], n_pages, self.page, self.kv_heads,
                            self.head_dim, k.stride(0), k.stride(1), k.stride(2))
        self._ref = ctypes.byref(self._kv)
        self._dtype = k.dtype

    def append(self, k, v, slots, stream=None):
        """tcb_kv_append: k and v [T, KV heads * head dim] (float32, float16 or
        bfloat16; parts of the projection's rows do), to slots int64 [T]."""
        T, n = k.shape
        _need(k.dtype is v.dtype and k.shape == v.shape and k.is_cuda and v.is_cuda, "k and v: two CUDA tensors of one shape and type are wanted")
        (ldk, uk), (ldv, uv) = k.stride(), v.stride()
        _need(n == self.kv_heads * self.head_dim and uk == 1 and uv == 1, "k and v: [T, KV heads * head dim] with dense rows is wanted")
        if k.dtype not in _TYPE:
            raise TcbError(2, "tcb_kv_append")
        rc = _lib().tcb_kv_append(self.ctx.handle, self._ref, T, k.data_ptr(), ldk if T > 1 else n, v.data_ptr(),
                                  ldv if T > 1 else n, _TYPE[k.dtype], _vec(slots, T, _I64, "slots"), _stream(self.ctx, stream))
        self.ctx._check(rc, "tcb_kv_append")

    def _q(self, q, out):
        if q.dtype != self._dtype or out.dtype != self._dtype:
            raise TcbError(2, "q and out are of the cache's type")
        _need(q.dim() == 3 and q.shape == out.shape and q.is_cuda and out.is_cuda, "q and out: [T, H, head dim] CUDA tensors are wanted")
        T, H, hd = q.shape
        _need(hd == self.head_dim, "q and out: the cache's head dim is wanted")
        for t in (q, out):
            _need(t.stride(2) == 1 and (H == 1 or t.stride(1) == hd), "q and out: dense heads are wanted")
        return T, H, q.data_ptr(), q.stride(0) if T > 1 else H * hd, out.data_ptr(), out.stride(0) if T > 1 else H * hd

    def attend(self, q, out, row_start, kv_len, tables, max_rows, max_len, scale=None, window=None, sinks=0, stream=None):
        """tcb_page_attn: q and out [T, H, head dim] in the cache's type;
        row_start int32 [B + 1], kv_len int32 [B], tables int32 [B, width];
        max_rows and max_len bound a request's rows and length; scale None is
        1 / sqrt(head dim), window None sees every earlier position."""
        T, H, qp, ldq, op, ldo = self._q(q, out)
        B = kv_len.shape[0]
        tp, width, ldt = _rows(tables, _I32, "tables")
        _need(tables.shape[0] >= B, "tables: a row per request is wanted")
        _need(window is None or window >= 0, "window: None or a whole number from 0 is wanted")
        rc = _lib().tcb_page_attn(self.ctx.handle, self._ref, B, T, H, qp, ldq, op, ldo,
                                  _vec(row_start, B + 1, _I32, "row_start"), _vec(kv_len, B, _I32, "kv_len"), tp, width,
                                  ldt, max_rows, max_len, 1.0 / math.sqrt(self.head_dim) if scale is None else scale,
                                  -1 if window is None else window, sinks, _stream(self.ctx, stream))
        self.ctx._check(rc, "tcb_page_attn")
        return out

    def attend_prefix(self, q, out, prefix, prefix_len, kv_len, tables, max_len, scale=None, stream=None):
        """tcb_prefix_attn: row b of q and out [B, H, head dim] is request b;
        prefix int32, the pages of the shared first prefix_len positions;
        kv_len int32 [B] counts them; tables int32 [B, width] as in attend."""
        T, H, qp, ldq, op, ldo = self._q(q, out)
        tp, width, ldt = _rows(tables, _I32, "tables")
        _need(tables.shape[0] >= T, "tables: a row per request is wanted")
        rc = _lib().tcb_prefix_attn(self.ctx.handle, self._ref, T, H, qp, ldq, op, ldo,
                                    _vec(prefix, -(-prefix_len // self.page), _I32, "prefix"), prefix_len,
                                    _vec(kv_len, T, _I32, "kv_len"), tp, width, ldt, max_len,
                                    1.0 / math.sqrt(self.head_dim) if scale is None else scale, _stream(self.ctx, stream))
        self.ctx._check(rc, "tcb_prefix_attn")
        return out


def penalize(ctx, logits, out, token=None, history=None, prompt_len=None, total_len=None, repetition=None,
             frequency=None, presence=None, bias_ids=None, bias=None, mask=None, mask_row=None, stream=None):
    """tcb_logits_penalize: logits [B, V] and out [B, V] (float32, float16 or
    bfloat16; out may be logits), token int64 [B] or None; history int64 [B,
    width] with prompt_len and total_len int32 [B]; repetition, frequency and
    presence float32 [B]; bias_ids int32 and bias float32 [B, n]; mask int32
    [masks, ceil(V / 32)], mask_row int32 [B]."""
    _need(logits.dim() == 2 and logits.shape == out.shape and logits.is_cuda and out.is_cuda, "logits and out: two [B, V] CUDA tensors are wanted")
    B, V = logits.shape
    for t in (logits, out):
        if t.dtype not in _TYPE:
            raise TcbError(2, "tcb_logits_penalize")
        _need(V <= 1 or t.stride(1) == 1, "logits and out: dense rows are wanted")
    f32 = torch.float32
    hp = width = ldh = 0
    if history is not None:
        hp, width, ldh = _rows(history, _I64, "history")
        _need(history.shape[0] >= B and total_len is not None, "history: a row per sequence and total_len are wanted")
    ip = vp = nb = ldb = 0
    if bias_ids is not None:
        ip, nb, ldb = _rows(bias_ids, _I32, "bias_ids")
        vp, nv, ldv = _rows(bias, f32, "bias")
        _need(nv == nb and ldv == ldb and bias_ids.shape[0] >= B and bias.shape[0] >= B, "bias_ids and bias: two tensors of one shape and stride are wanted")
    mp = nm = ldm = 0
    if mask is not None:
        mp, words, ldm = _rows(mask, _I32, "mask")
        nm = mask.shape[0]
        _need(words >= -(-V // 32) and (mask_row is not None or nm >= B), "mask: ceil(V / 32) words in a row, and a row per sequence or mask_row, are wanted")
    a = _LogitsArgs(B, V, logits.data_ptr(), _TYPE[logits.dtype], logits.stride(0) if B > 1 else V,
                    out.data_ptr(), _TYPE[out.dtype], out.stride(0) if B > 1 else V,
                    _vec(token, B, _I64, "token") if token is not None else 0, hp, width, ldh,
                    _vec(prompt_len, B, _I32, "prompt_len") if prompt_len is not None else 0,
                    _vec(total_len, B, _I32, "total_len") if total_len is not None else 0,
                    _vec(repetition, B, f32, "repetition") if repetition is not None else 0,
                    _vec(frequency, B, f32, "frequency") if frequency is not None else 0,
                    _vec(presence, B, f32, "presence") if presence is not None else 0,
                    ip, vp, nb, ldb, mp, nm, ldm,
                    _vec(mask_row, B, _I32, "mask_row") if mask_row is not None else 0)
    rc = _lib().tcb_logits_penalize(ctx.handle, ctypes.byref(a), _stream(ctx, stream))
    ctx._check(rc, "tcb_logits_penalize")
    return out
