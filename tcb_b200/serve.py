"""Serving operators over a paged K/V cache (include/tcb.h, tcb_page_* and
tcb_logits_penalize): a thin view for torch CUDA tensors (the checks and the
call itself are in tcb_b200/csrc/tcb_torch.cpp; the C structures and argument
types are here).

One step of a batch of requests:
  plan(...)             pages, row offsets, slots and positions of the step
  Pages.append(...)     the step's K/V rows into the cache
  Pages.attend(...)     causal attention over the pages, with a sliding
                        window and first positions that stay visible
  Pages.attend_prefix(...)  a decode step of a batch over one shared prefix
  penalize(...)         penalties, biases and masks on the logits, the pick
All lengths and page numbers are int32 tensors on the device; nothing here
waits for the device.  Every call runs on `stream` (the current one when it is
None), and calls on one context are to be ordered on one stream; tensors given
to another stream than their own are the caller's to keep until it is done.
Device-side findings (a page outside the pool, a length past max_len) are read with
Context.device_error().
"""
from __future__ import annotations

import ctypes
import os

import torch

from . import BF16, F16, HERE, TcbError, lib

_TYPE = {torch.float16: F16, torch.bfloat16: BF16}


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


_torch_view = None


def _view():
    """The module _tcb_torch (tcb_b200/csrc/tcb_torch.cpp), bound to the loaded
    library.  No fallback: a missing module raises."""
    global _torch_view
    if _torch_view is None:
        path = os.path.join(HERE, "_tcb_torch.so")
        if not os.path.exists(path):
            raise ImportError(f"{path} is missing; build it with `python -m tcb_b200.build`")
        from . import _tcb_torch as m

        L = _lib()
        m.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (L.tcb_page_plan, L.tcb_kv_append, L.tcb_page_attn,
                                                                L.tcb_prefix_attn, L.tcb_logits_penalize)))
        _torch_view = m
    return _torch_view


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def plan(ctx, page, cached, fresh, tables, free, n_free, row_start, kv_len, slots, positions, balance, taken=None,
         stream=None):
    """tcb_page_plan: cached and fresh int32 [B]; tables int32 [B, width]
    (extended in place); free int32, the stack of free pages, of which the
    first n_free[0] are free; written: row_start int32 [B + 1], kv_len int32
    [B], slots int64 and positions int32 [rows], taken int32 [1] or None (the
    pages taken, by which the caller lowers n_free) and balance int32 [1] (n_free
    less taken; or, below 0, the pages that were short, where a request that lacks
    none is served behind refused ones).  A refused request has kv_len 0.  Outputs
    that overlap an input, the tables or one another raise TcbError."""
    rc = _view().plan(ctx.handle.value, ctx.device, page, cached, fresh, tables, free, n_free, row_start, kv_len, slots,
                      positions, balance, taken, stream)
    if rc:
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
        self._at = ctypes.addressof(self._kv)
        _need(k.device.index == ctx.device, "k and v: tensors of the context's device are wanted")

    def append(self, k, v, slots, stream=None):
        """tcb_kv_append: k and v [T, KV heads * head dim] (float32, float16 or
        bfloat16; parts of the projection's rows do), to slots int64 [T]."""
        rc = _view().append(self.ctx.handle.value, self.ctx.device, self._at, k, v, slots, stream)
        if rc:
            self.ctx._check(rc, "tcb_kv_append")

    def attend(self, q, out, row_start, kv_len, tables, max_rows, max_len, scale=None, window=None, sinks=0, stream=None):
        """tcb_page_attn: q and out [T, H, head dim] in the cache's type;
        row_start int32 [B + 1], kv_len int32 [B], tables int32 [B, width];
        max_rows and max_len bound a request's rows and length; scale None is
        1 / sqrt(head dim), window None sees every earlier position."""
        rc = _view().attend(self.ctx.handle.value, self.ctx.device, self._at, q, out, row_start, kv_len, tables, max_rows,
                            max_len, scale, window, sinks, stream)
        if rc:
            self.ctx._check(rc, "tcb_page_attn")
        return out

    def attend_prefix(self, q, out, prefix, prefix_len, kv_len, tables, max_len, scale=None, stream=None):
        """tcb_prefix_attn: row b of q and out [B, H, head dim] is request b;
        prefix int32, the pages of the shared first prefix_len positions;
        kv_len int32 [B] counts them; tables int32 [B, width] as in attend."""
        rc = _view().attend_prefix(self.ctx.handle.value, self.ctx.device, self._at, q, out, prefix, prefix_len, kv_len,
                                   tables, max_len, scale, stream)
        if rc:
            self.ctx._check(rc, "tcb_prefix_attn")
        return out


def penalize(ctx, logits, out, token=None, history=None, prompt_len=None, total_len=None, repetition=None,
             frequency=None, presence=None, bias_ids=None, bias=None, mask=None, mask_row=None, stream=None):
    """tcb_logits_penalize: logits [B, V] and out [B, V] (float32, float16 or
    bfloat16; out may be logits), token int64 [B] or None; history int64 [B,
    width] with prompt_len and total_len int32 [B]; repetition, frequency and
    presence float32 [B]; bias_ids int32 and bias float32 [B, n]; mask int32
    [masks, ceil(V / 32)], mask_row int32 [B]."""
    rc = _view().penalize(ctx.handle.value, ctx.device, logits, out, token, history, prompt_len, total_len, repetition,
                          frequency, presence, bias_ids, bias, mask, mask_row, stream)
    if rc:
        ctx._check(rc, "tcb_logits_penalize")
    return out
