"""Serving: a paged 8-bit key/value cache and the operators that work on it.

The reference recomputes a sequence's whole prefix for every token it adds
(sparse_attention.py:1420-1510 takes the full x); a program that generates
text keeps the keys and values instead.  Here they live in pages of 32, 64 or
128 tokens as e4m3 codes, with a power-of-two scale per page and kv head:

* :func:`plan_pages` -- block tables, slots and positions of a ragged batch
  from its requests' lengths, on the GPU (:class:`PageTable` keeps the tables
  of a running server and calls it);
* :func:`cache_append` -- the batch's keys and values into the cache;
* :func:`select_pages` -- per row and kv head the pages whose bound ranks
  first: the paged counterpart of the neighbour graph's self / window / global
  / best-scored union;
* :func:`cached_attention` -- attention over every earlier key, or over the
  selected pages.

All are inference only and run on ROCm devices only; none synchronises with
the host, so a whole step can be captured into a HIP graph.
"""
from __future__ import annotations

import contextlib
import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib

E4M3 = torch.float8_e4m3fn
PAGE_SIZES = (32, 64, 128)
MAX_HEAD_DIM = 256


def store_dim(d_head: int) -> int:
    """Head dim the cache stores rows of d_head numbers at: 64, 128 or 256."""
    if not 1 <= d_head <= MAX_HEAD_DIM:
        raise RuntimeError(f"ssa_amd: head dim {d_head} unsupported by the cache "
                           f"(1..{MAX_HEAD_DIM})")
    return 64 if d_head <= 64 else 128 if d_head <= 128 else 256


def _need(cond, what, msg):
    if not cond:
        raise RuntimeError(f"ssa_amd.{what}: {msg}")


def _ints(t, name, shape, what, dtype=torch.int32):
    """Raise unless t is a contiguous integer tensor of this shape."""
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise RuntimeError(f"ssa_amd.{what}: {name} must be a contiguous {dtype} tensor of shape "
                           f"{tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def _one_device(what, dev, *tensors):
    if dev.type != "cuda":
        raise RuntimeError(f"ssa_amd.{what} runs on ROCm devices only (got a tensor on {dev})")
    for t in tensors:
        if t.device != dev:
            raise RuntimeError(f"ssa_amd.{what}: tensors on {dev} and {t.device}")


def _inference(what, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"ssa_amd.{what} is inference only: call it under torch.no_grad()")


def _on(dev):
    """The device made current for a launch (nothing to do where it is)."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


# ---------------------------------------------------------------------------- cache
class PagedKVCache:
    """One layer's keys and values in `num_pages` pages of `page_size` tokens.

    k_codes (pages, n_kv, page, D) and v_codes (pages, n_kv, D, page) e4m3,
    bounds (pages, n_kv, 2, D) e4m3 (per channel the smallest and largest key
    code of the page), k_scale and v_scale (pages, n_kv) fp32 powers of two; D
    = :func:`store_dim` (d_head).  A number is code * scale.
    """

    def __init__(self, num_pages: int, num_kv_heads: int, d_head: int, page_size: int = 64,
                 device="cuda"):
        D = store_dim(d_head)
        z = dict(dtype=torch.uint8, device=device)
        one = dict(dtype=torch.float32, device=device)
        self._set(torch.zeros((num_pages, num_kv_heads, page_size, D), **z).view(E4M3),
                  torch.zeros((num_pages, num_kv_heads, D, page_size), **z).view(E4M3),
                  torch.zeros((num_pages, num_kv_heads, 2, D), **z).view(E4M3),
                  torch.ones((num_pages, num_kv_heads), **one),
                  torch.ones((num_pages, num_kv_heads), **one), d_head)

    @classmethod
    def from_tensors(cls, k_codes, v_codes, bounds, k_scale, v_scale,
                     d_head: int) -> "PagedKVCache":
        """A cache over buffers the caller holds (contiguous, laid out as above;
        value codes free of NaN)."""
        self = cls.__new__(cls)
        self._set(k_codes, v_codes, bounds, k_scale, v_scale, d_head)
        return self

    def _set(self, k_codes, v_codes, bounds, k_scale, v_scale, d_head):
        what, D = "PagedKVCache", store_dim(d_head)
        _need(k_codes.dim() == 4 and k_codes.shape[3] == D, what,
              f"k_codes {tuple(k_codes.shape)} are not (pages, kv heads, page, {D})")
        P, H, ps, _ = k_codes.shape
        _need(P >= 1 and H >= 1 and ps in PAGE_SIZES, what,
              f"{P} pages of {ps} tokens, {H} kv heads (pages of 32, 64 or 128 tokens)")
        for t, shape, name in ((k_codes, (P, H, ps, D), "k_codes"),
                               (v_codes, (P, H, D, ps), "v_codes"),
                               (bounds, (P, H, 2, D), "bounds")):
            if t.shape != shape or t.dtype != E4M3 or not t.is_contiguous():
                raise RuntimeError(f"ssa_amd.{what}: {name} must be contiguous {E4M3} {shape}, "
                                   f"got {t.dtype} {tuple(t.shape)}")
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if t.shape != (P, H) or t.dtype != torch.float32 or not t.is_contiguous():
                raise RuntimeError(f"ssa_amd.{what}: {name} must be contiguous float32 {(P, H)}, "
                                   f"got {t.dtype} {tuple(t.shape)}")
        dev = k_codes.device
        for t in (v_codes, bounds, k_scale, v_scale):
            _need(t.device == dev, what, f"buffers on {dev} and {t.device}")
        self.k_codes, self.v_codes, self.bounds = k_codes, v_codes, bounds
        self.k_scale, self.v_scale = k_scale, v_scale
        self.num_pages, self.num_kv_heads, self.page_size, self.d_head = P, H, ps, d_head
        self.device = dev
        self._c = _lib.KVCacheStruct(k_codes.data_ptr(), v_codes.data_ptr(), bounds.data_ptr(),
                                     k_scale.data_ptr(), v_scale.data_ptr(), P, H, ps, D, d_head)


# ---------------------------------------------------------------------------- plan
@dataclass
class PagePlan:
    """Where a ragged batch's rows stand.  Request r's rows are starts[r] ..
    starts[r + 1] - 1; rows of no request (padding, a refused request) have
    request, position and slot -1.  The last four are what :func:`plan_pages`
    says besides what the attention needs."""
    block_table: torch.Tensor                    # (R, width) int32
    starts: torch.Tensor                         # (R + 1,) int32
    requests: torch.Tensor                       # (T,) int32
    positions: torch.Tensor                      # (T,) int32
    slots: Optional[torch.Tensor] = None         # (T,) int64: page * page_size + offset
    lengths: Optional[torch.Tensor] = None       # (R,) int32: tokens after the batch
    free_count: Optional[torch.Tensor] = None    # (1,) int32: pages left
    refused: Optional[torch.Tensor] = None       # (1,) int32: requests refused


def plan_pages(cached, new_rows, block_table, free_pages, free_count, *, page_size: int,
               num_rows: int) -> PagePlan:
    """Block tables, slots and positions of a batch of `num_rows` rows.

    cached, new_rows (R,) int32: tokens each request holds and rows it brings;
    block_table (R, width) int32, unit last stride, takes the new pages in
    place; free_pages int32: a stack whose top is free_pages[free_count - 1]
    (free_count (1,) int32; the new count is returned, not written).  A request
    is refused, as a whole, when its rows pass num_rows, its tokens pass width
    pages, a length is negative, or the free pages do not reach it."""
    what = "plan_pages"
    _need(cached.dim() == 1 and block_table.dim() == 2 and free_pages.dim() == 1, what,
          f"cached {tuple(cached.shape)}, block_table {tuple(block_table.shape)}, free_pages "
          f"{tuple(free_pages.shape)}")
    R, width = block_table.shape
    _need(R >= 1 and width >= 1 and num_rows >= 0, what,
          f"{R} requests of {width} pages, {num_rows} rows")
    _ints(cached, "cached", (R,), what)
    _ints(new_rows, "new_rows", (R,), what)
    _ints(free_pages, "free_pages", free_pages.shape, what)
    _ints(free_count, "free_count", (1,), what)
    _need(block_table.dtype == torch.int32 and block_table.stride(1) == 1
          and (R == 1 or block_table.stride(0) >= width), what,
          f"block_table must be int32 rows of unit stride, got {block_table.dtype} strides "
          f"{block_table.stride()}")
    dev = cached.device
    _one_device(what, dev, new_rows, block_table, free_pages, free_count)
    T = int(num_rows)
    buf = torch.empty(2 * T + 2 * R + 3, dtype=torch.int32, device=dev)
    starts, lengths, positions, requests, count, refused = buf.split_with_sizes(
        (R + 1, R, T, T, 1, 1))
    slots = torch.empty(T, dtype=torch.int64, device=dev)
    p = buf.data_ptr()
    a = _lib.PagePlanArgs(
        cached.data_ptr(), new_rows.data_ptr(), block_table.data_ptr(),
        max(block_table.stride(0), width), R, width, page_size, T, free_pages.data_ptr(),
        free_pages.numel(), free_count.data_ptr(), p, p + 4 * (R + 1), slots.data_ptr(),
        p + 4 * (2 * R + 1), p + 4 * (2 * R + 1 + T), p + 4 * (2 * R + 1 + 2 * T),
        p + 4 * (2 * R + 2 + 2 * T))
    with _on(dev):
        _lib._check(_lib.lib().ssa_page_plan(ctypes.byref(a), _lib._stream(cached)), what)
    return PagePlan(block_table, starts, requests, positions, slots, lengths, count, refused)


class PageTable:
    """The block tables of a running server: `max_requests` places of up to
    `max_pages` pages each out of `num_pages`, shared by all layers' caches.
    Its tensors keep their addresses, so a captured step can be replayed."""

    def __init__(self, max_requests: int, max_pages: int, num_pages: int, page_size: int = 64,
                 device="cuda"):
        z = dict(dtype=torch.int32, device=device)
        _need(page_size in PAGE_SIZES, "PageTable", f"pages of {page_size} tokens (32, 64 or 128)")
        self.page_size, self.num_pages = page_size, num_pages
        self.block_table = torch.full((max_requests, max_pages), -1, **z)
        self.lengths = torch.zeros(max_requests, **z)
        # page 0 on top; one entry more takes what release() has no page for
        self._free = torch.arange(num_pages - 1, -2, -1, **z)
        self.free_count = torch.full((1,), num_pages, **z)

    def plan(self, new_rows: torch.Tensor, num_rows: int) -> PagePlan:
        """:func:`plan_pages` for the places' current lengths, which then count
        the admitted rows."""
        p = plan_pages(self.lengths, new_rows, self.block_table, self._free[:self.num_pages],
                       self.free_count, page_size=self.page_size, num_rows=num_rows)
        self.lengths.copy_(p.lengths)
        self.free_count.copy_(p.free_count)
        return p

    def release(self, places: torch.Tensor) -> None:
        """Give the pages of these places (integer tensor) back and empty them."""
        R, W = self.block_table.shape
        gone = torch.zeros(R, dtype=torch.bool, device=self.lengths.device)
        gone[places.to(self.lengths.device, torch.int64)] = True
        held = (self.lengths + self.page_size - 1) // self.page_size
        col = torch.arange(W, device=self.lengths.device)
        give = (gone[:, None] & (col < held[:, None])).reshape(-1)
        at = torch.where(give, self.free_count + torch.cumsum(give, 0) - 1, self.num_pages)
        self._free[at] = self.block_table.reshape(-1)
        self.free_count += give.sum(dtype=torch.int32)
        self.block_table.masked_fill_(gone[:, None], -1)
        self.lengths.masked_fill_(gone, 0)


# ---------------------------------------------------------------------------- append
def _rows3(t, name, what):
    _need(t.dim() == 3, what, f"{name} must be 3-D (rows, heads, d), got {tuple(t.shape)}")
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def cache_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Write k and v (T, n_kv, d_head; float32, bfloat16 or float16) into the
    cache at `slots` (T,) int64 (page * page_size + offset; outside the cache:
    skipped).  The rows of one page are adjacent and ascend by one, as
    :func:`plan_pages` makes them.

    Where a page's scale has to grow for them, its earlier codes are rounded to
    the new one.  A row with a NaN, an infinity or a magnitude of 2^120 or more
    makes every later query that sees it NaN."""
    what = "cache_append"
    k, v = _rows3(k, "k", what), _rows3(v, "v", what)
    T, H, d = k.shape
    _need(v.shape == k.shape and v.dtype == k.dtype, what,
          f"k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} differ")
    _need(H == cache.num_kv_heads and d == cache.d_head, what,
          f"rows of {H} heads of dim {d} into a cache of {cache.num_kv_heads} of dim "
          f"{cache.d_head}")
    _ints(slots, "slots", (T,), what, torch.int64)
    _inference(what, k, v)
    dt = _lib.dtype_code(k.dtype)
    _one_device(what, k.device, v, slots, cache.k_codes)
    a = _lib.CacheAppendArgs(cache._c, k.data_ptr(), v.data_ptr(), dt, T, k.stride(0), k.stride(1),
                             v.stride(0), v.stride(1), slots.data_ptr())
    with _on(k.device):
        _lib._check(_lib.lib().ssa_cache_append(ctypes.byref(a), _lib._stream(k)), what)


# ---------------------------------------------------------------------------- select, attend
def _batch(what, q, cache, plan):
    """Checked (q, ssa_batch_rows) of a batch."""
    q = _rows3(q, "q", what)
    T, Hq, d = q.shape
    _need(Hq >= 1 and Hq % cache.num_kv_heads == 0, what,
          f"{Hq} query heads are not a multiple of {cache.num_kv_heads} kv heads")
    _need(d == cache.d_head, what, f"q has head dim {d}, the cache {cache.d_head}")
    bt = plan.block_table
    _need(bt.dim() == 2 and bt.shape[0] >= 1 and bt.shape[1] >= 1, what,
          f"block_table {tuple(bt.shape)}")
    R, width = bt.shape
    _need(bt.dtype == torch.int32 and bt.stride(1) == 1 and (R == 1 or bt.stride(0) >= width),
          what, f"block_table must be int32 rows of unit stride, got {bt.dtype} strides "
          f"{bt.stride()}")
    _ints(plan.starts, "starts", (R + 1,), what)
    _ints(plan.requests, "requests", (T,), what)
    _ints(plan.positions, "positions", (T,), what)
    _inference(what, q)
    _one_device(what, q.device, bt, plan.starts, plan.requests, plan.positions, cache.k_codes)
    return q, _lib.BatchRows(bt.data_ptr(), max(bt.stride(0), width), R, width,
                             plan.starts.data_ptr(), plan.requests.data_ptr(),
                             plan.positions.data_ptr(), T)


def select_pages(q: torch.Tensor, cache: PagedKVCache, plan: PagePlan, top_k: int, *,
                 first: int = 1, recent: int = 1) -> torch.Tensor:
    """(T, n_kv, top_k) int32: the pages of its request each row of q (T, Hq,
    d_head) should attend to, per kv head, in ascending order, -1 behind the
    last: the `first` ones, the `recent` ones up to the row's own, and of the
    others those with the largest bound of the group's summed scores (ties to
    the lower page).  recent >= 1, first + recent <= top_k."""
    what = "select_pages"
    _need(first >= 0 and recent >= 1 and first + recent <= top_k, what,
          f"first={first} recent={recent} top_k={top_k} (recent >= 1, both within top_k)")
    q, rows = _batch(what, q, cache, plan)
    T, Hq, _ = q.shape
    out = torch.empty((T, cache.num_kv_heads, top_k), dtype=torch.int32, device=q.device)
    a = _lib.SelectPagesArgs(cache._c, rows, q.data_ptr(), _lib.dtype_code(q.dtype), Hq,
                             q.stride(0), q.stride(1), top_k, first, recent, out.data_ptr())
    with _on(q.device):
        _lib._check(_lib.lib().ssa_select_pages(ctypes.byref(a), _lib._stream(q)), what)
    return out


def cached_attention(q: torch.Tensor, cache: PagedKVCache, plan: PagePlan, *,
                     scale: Optional[float] = None, pages: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of q (T, Hq, d_head) over its requests' cached keys up
    to each row's own position, or over `pages` (T, n_kv, top) int32 of them
    (negative: none; each page at most once).  scale: 1 / sqrt(d_head) unless
    given.  Query head h reads kv head h // (Hq // n_kv).  Rows that see no key
    (padding, a refused request) get zeros.  Returns (T, Hq, d_head) in q's
    dtype (`out`, where given)."""
    what = "cached_attention"
    q, rows = _batch(what, q, cache, plan)
    T, Hq, d = q.shape
    top, pp = 0, None
    if pages is not None:
        _need(pages.dim() == 3 and pages.shape[2] >= 1, what, f"pages {tuple(pages.shape)}")
        top = pages.shape[2]
        _ints(pages, "pages", (T, cache.num_kv_heads, top), what)
        _one_device(what, q.device, pages)
        pp = pages.data_ptr()
    if out is None:
        out = torch.empty((T, Hq, d), dtype=q.dtype, device=q.device)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device
              and (out.stride(2) == 1 or d == 1), what,
              f"out {out.dtype} {tuple(out.shape)} does not fit q {q.dtype} {tuple(q.shape)}")
    a = _lib.CachedAttentionArgs(cache._c, rows, q.data_ptr(), out.data_ptr(),
                                 _lib.dtype_code(q.dtype), Hq, q.stride(0), q.stride(1),
                                 out.stride(0), out.stride(1),
                                 d ** -0.5 if scale is None else float(scale), pp, top)
    L = _lib.lib()
    with _on(q.device):
        n = L.ssa_cached_attention_workspace_bytes(ctypes.byref(a))
        if n < 0:
            _lib._check(int(n), what)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        _lib._check(L.ssa_cached_attention(ctypes.byref(a), None if ws is None else ws.data_ptr(),
                                           n, _lib._stream(q)), what)
    return out
