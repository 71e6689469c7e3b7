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
the host, so a whole step (:meth:`PageTable.plan` and these) can be captured
into a HIP graph.
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


# The checks below run on every call of a few microseconds: messages are formed only
# where one fails.
def _refuse(what, msg):
    raise RuntimeError(f"ssa_amd.{what}: {msg}")


def _ints(t, name, shape, what, dtype=torch.int32):
    """Raise unless t is a contiguous integer tensor of this shape."""
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        _refuse(what, f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, got "
                f"{t.dtype} {tuple(t.shape)}")


def _table(bt, what):
    """(R, width, elements between rows) of a block table."""
    if bt.dim() != 2 or bt.dtype != torch.int32:
        _refuse(what, f"block_table must be 2-D int32, got {bt.dtype} {tuple(bt.shape)}")
    (R, width), (step, unit) = bt.shape, bt.stride()
    if R < 1 or width < 1 or (unit != 1 and width > 1) or (step < width and R > 1):
        _refuse(what, f"block_table {tuple(bt.shape)} must have rows of unit stride, got strides "
                f"{bt.stride()}")
    return R, width, step if step > width else width


def _one_device(what, dev, *tensors):
    if dev.type != "cuda":
        raise RuntimeError(f"ssa_amd.{what} runs on ROCm devices only (got a tensor on {dev})")
    for t in tensors:
        if t.device != dev:
            raise RuntimeError(f"ssa_amd.{what}: tensors on {dev} and {t.device}")


def _inference(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                _refuse(what, "inference only: call it under torch.no_grad()")


_HERE = contextlib.nullcontext()


def _on(dev):
    """The device made current for a launch (nothing to do where it is)."""
    i = dev.index
    return _HERE if i is None or i == torch.cuda.current_device() else torch.cuda.device(dev)


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
        if k_codes.dim() != 4 or k_codes.shape[3] != D:
            _refuse(what, f"k_codes {tuple(k_codes.shape)} are not (pages, kv heads, page, {D})")
        P, H, ps, _ = k_codes.shape
        if P < 1 or H < 1 or ps not in PAGE_SIZES:
            _refuse(what, f"{P} pages of {ps} tokens, {H} kv heads (pages of 32, 64 or 128 tokens)")
        dev, n = k_codes.device, (P, H)
        for t, shape, dt, name in ((k_codes, (P, H, ps, D), E4M3, "k_codes"),
                                   (v_codes, (P, H, D, ps), E4M3, "v_codes"),
                                   (bounds, (P, H, 2, D), E4M3, "bounds"),
                                   (k_scale, n, torch.float32, "k_scale"),
                                   (v_scale, n, torch.float32, "v_scale")):
            if t.shape != shape or t.dtype != dt or t.device != dev or not t.is_contiguous():
                _refuse(what, f"{name} must be contiguous {dt} {shape} on {dev}, got {t.dtype} "
                        f"{tuple(t.shape)} on {t.device}")
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
    R, width, step = _table(block_table, what)
    if not 0 <= num_rows < 1 << 31:
        _refuse(what, f"{num_rows} rows (0 to 2^31 - 1)")
    _ints(cached, "cached", (R,), what)
    _ints(new_rows, "new_rows", (R,), what)
    if free_pages.dim() != 1:
        _refuse(what, f"free_pages {tuple(free_pages.shape)}")
    _ints(free_pages, "free_pages", free_pages.shape, what)
    _ints(free_count, "free_count", (1,), what)
    dev = cached.device
    _one_device(what, dev, new_rows, block_table, free_pages, free_count)
    T = int(num_rows)
    slots = torch.empty(T, dtype=torch.int64, device=dev)
    buf = slots.new_empty(2 * T + 2 * R + 3, dtype=torch.int32)
    starts, lengths, positions, requests, count, refused = buf.split_with_sizes(
        (R + 1, R, T, T, 1, 1))
    p = buf.data_ptr()
    q = p + 4 * (2 * R + 1)
    a = _lib.PagePlanArgs(
        cached.data_ptr(), new_rows.data_ptr(), block_table.data_ptr(), step, R, width, page_size,
        T, free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), p, p + 4 * (R + 1),
        slots.data_ptr(), q, q + 4 * T, q + 8 * T, q + 8 * T + 4)
    with _on(dev):
        rc = _lib.lib().ssa_page_plan(ctypes.byref(a), _lib._stream(cached))
    if rc:
        _lib._check(rc, what)
    return PagePlan(block_table, starts, requests, positions, slots, lengths, count, refused)


class PageTable:
    """The block tables of a running server: `max_requests` places of up to
    `max_pages` pages each out of `num_pages`, shared by all layers' caches.
    Its tensors keep their addresses, so a captured step can be replayed."""

    def __init__(self, max_requests: int, max_pages: int, num_pages: int, page_size: int = 64,
                 device="cuda"):
        z = dict(dtype=torch.int32, device=device)
        if page_size not in PAGE_SIZES:
            _refuse("PageTable", f"pages of {page_size} tokens (32, 64 or 128)")
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
        """Give the pages of these places (integer tensor; what names no place is
        passed over) back and empty them.  Between a captured step's replays, not in
        a graph itself (its torch operations are not made for that)."""
        R, W = self.block_table.shape
        places = places.to(self.lengths.device, torch.int64).reshape(1, -1)
        gone = (torch.arange(R, device=self.lengths.device)[:, None] == places).any(1)
        held = (self.lengths + self.page_size - 1) // self.page_size
        col = torch.arange(W, device=self.lengths.device)
        give = (gone[:, None] & (col < held[:, None])).reshape(-1)
        upto = torch.cumsum(give, 0)
        at = torch.where(give, self.free_count + upto - 1, self.num_pages)
        self._free[at] = self.block_table.reshape(-1)
        self.free_count += upto[-1]
        self.block_table.masked_fill_(gone[:, None], -1)
        self.lengths.masked_fill_(gone, 0)


# ---------------------------------------------------------------------------- append
def _rows3(t, name, what):
    if t.dim() != 3 or t.shape[0] >= 1 << 31:
        _refuse(what, f"{name} must be 3-D (rows, heads, d) of less than 2^31 rows, got "
                f"{tuple(t.shape)}")
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
    dt = k.dtype
    if v.shape != k.shape or v.dtype != dt:
        _refuse(what, f"k {dt} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} differ")
    if H != cache.num_kv_heads or d != cache.d_head:
        _refuse(what, f"rows of {H} heads of dim {d} into a cache of {cache.num_kv_heads} of dim "
                f"{cache.d_head}")
    _ints(slots, "slots", (T,), what, torch.int64)
    _inference(what, k, v)
    code = _lib.dtype_code(dt)
    dev = k.device
    _one_device(what, dev, v, slots, cache.k_codes)
    (k_st, k_sh, _), (v_st, v_sh, _) = k.stride(), v.stride()
    a = _lib.CacheAppendArgs(cache._c, k.data_ptr(), v.data_ptr(), code, T, k_st, k_sh, v_st, v_sh,
                             slots.data_ptr())
    with _on(dev):
        rc = _lib.lib().ssa_cache_append(ctypes.byref(a), _lib._stream(k))
    if rc:
        _lib._check(rc, what)


# ---------------------------------------------------------------------------- select, attend
def _batch(what, q, cache, plan):
    """Checked (q, ssa_batch_rows, T, Hq, d) of a batch."""
    q = _rows3(q, "q", what)
    T, Hq, d = q.shape
    if Hq < 1 or Hq % cache.num_kv_heads or d != cache.d_head:
        _refuse(what, f"q has {Hq} heads of dim {d}, the cache {cache.num_kv_heads} of dim "
                f"{cache.d_head} (query heads a multiple of kv heads, one head dim)")
    bt, starts, requests, positions = plan.block_table, plan.starts, plan.requests, plan.positions
    R, width, step = _table(bt, what)
    _ints(starts, "starts", (R + 1,), what)
    _ints(requests, "requests", (T,), what)
    _ints(positions, "positions", (T,), what)
    _inference(what, q)
    _one_device(what, q.device, bt, starts, requests, positions, cache.k_codes)
    return q, _lib.BatchRows(bt.data_ptr(), step, R, width, starts.data_ptr(), requests.data_ptr(),
                             positions.data_ptr(), T), T, Hq, d


def select_pages(q: torch.Tensor, cache: PagedKVCache, plan: PagePlan, top_k: int, *,
                 first: int = 1, recent: int = 1) -> torch.Tensor:
    """(T, n_kv, top_k) int32: the pages of its request each row of q (T, Hq,
    d_head) should attend to, per kv head, in ascending order, -1 behind the
    last: the `first` ones, the `recent` ones up to the row's own, and of the
    others those with the largest bound of the group's summed scores (ties to
    the lower page).  recent >= 1, first + recent <= top_k."""
    what = "select_pages"
    if not (first >= 0 and recent >= 1 and first + recent <= top_k):
        _refuse(what, f"first={first} recent={recent} top_k={top_k} (recent >= 1, both within "
                "top_k)")
    q, rows, T, Hq, _ = _batch(what, q, cache, plan)
    out = torch.empty((T, cache.num_kv_heads, top_k), dtype=torch.int32, device=q.device)
    q_st, q_sh, _ = q.stride()
    a = _lib.SelectPagesArgs(cache._c, rows, q.data_ptr(), _lib.dtype_code(q.dtype), Hq, q_st, q_sh,
                             top_k, first, recent, out.data_ptr())
    with _on(q.device):
        rc = _lib.lib().ssa_select_pages(ctypes.byref(a), _lib._stream(q))
    if rc:
        _lib._check(rc, what)
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
    q, rows, T, Hq, d = _batch(what, q, cache, plan)
    dev = q.device
    top, pp = 0, None
    if pages is not None:
        if pages.dim() != 3 or pages.shape[2] < 1:
            _refuse(what, f"pages {tuple(pages.shape)} are not (rows, kv heads, pages)")
        top = pages.shape[2]
        _ints(pages, "pages", (T, cache.num_kv_heads, top), what)
        _one_device(what, dev, pages)
        pp = pages.data_ptr()
    if out is None:
        out = torch.empty((T, Hq, d), dtype=q.dtype, device=dev)
    elif (out.shape != q.shape or out.dtype != q.dtype or out.device != dev
          or (out.stride(2) != 1 and d > 1)):
        _refuse(what, f"out {out.dtype} {tuple(out.shape)} strides {out.stride()} does not fit q "
                f"{q.dtype} {tuple(q.shape)}")
    (q_st, q_sh, _), (o_st, o_sh, _) = q.stride(), out.stride()
    a = _lib.CachedAttentionArgs(cache._c, rows, q.data_ptr(), out.data_ptr(),
                                 _lib.dtype_code(q.dtype), Hq, q_st, q_sh, o_st, o_sh,
                                 d ** -0.5 if scale is None else float(scale), pp, top)
    L, ref = _lib.lib(), ctypes.byref(a)
    with _on(dev):
        n = L.ssa_cached_attention_workspace_bytes(ref)
        if n < 0:
            _lib._check(int(n), what)
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        rc = L.ssa_cached_attention(ref, ws.data_ptr() if n else None, n, _lib._stream(q))
    if rc:
        _lib._check(rc, what)
    return out
