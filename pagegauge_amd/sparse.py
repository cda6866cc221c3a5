"""Attention over the part of a long history that matters to a token.

Of each request's INT8 pages, every KV head reads a fixed number, picked for the
query by a cheap score:

* ``allocate_bounds`` -- int8 [pages, Hkv, 2, 128] beside a pool: the least and the
  largest K code of each channel of a page, a sixteenth of the page's bytes;
* ``key_bounds`` -- taken from the codes of pages as they are completed, by a prompt
  or by a step;
* ``SelectedPagesDecode.select`` -- the score of a page is the largest product that
  a key within its bounds could have with a query head of the KV head, in whole
  numbers (``include/pagegauge_hip.h`` states it to the bit); the highest are
  picked, the first and last pages of the table always;
* ``SelectedPagesDecode.run`` -- attention over the picked pages, an exact FP16 tail
  and the value center.

Everything runs on the current stream and nothing but ``plan`` synchronises (and checks
of page ids, as ``prefix`` says).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _capi
from .decode import _check_query, _check_scale, _num_cus
from .prefix import DIM, PAGE, _SegmentDecode, _ptr, _tables

_BOUNDS = "bounds must be contiguous int8 [pages,Hkv,2,128]"


def allocate_bounds(pages: int, kv_heads: int, device="cuda") -> torch.Tensor:
    """The bounds of a pool, zeroed."""
    return torch.zeros(pages, kv_heads, 2, DIM, dtype=torch.int8, device=device)


def key_bounds(key_codes: torch.Tensor, bounds: torch.Tensor, *, page_ids: Optional[torch.Tensor] = None,
               lengths: Optional[torch.Tensor] = None) -> None:
    """Write the bounds of pages ``page_ids`` (device int32 [n]; None: the whole pool)
    of ``key_codes`` int8 [pages, 16, Hkv, 128] into ``bounds`` [pages, Hkv, 2, 128].
    ``lengths`` (device int32 [n]) is the tokens that each page holds, 16 if not given;
    a page without tokens gets 127 and -128, whose score is the lowest that bounds under
    the same K scale (above 0) can have: a page that was never written and has a scale of 0
    scores 0.  Ids outside the pool (-1) are skipped; the others must differ from each
    other."""
    if key_codes.dim() != 4 or key_codes.shape[2] == 0:
        raise ValueError("key_codes must be contiguous int8 [pages,16,Hkv,128]")
    pages, _, heads, _ = key_codes.shape
    device = key_codes.get_device()
    codes_at = _capi.pointer(key_codes, torch.int8, (pages, PAGE, heads, DIM), device,
                             "key_codes must be contiguous int8 [pages,16,Hkv,128]")
    bounds_at = _capi.pointer(bounds, torch.int8, (pages, heads, 2, DIM), device, _BOUNDS)
    count = pages if page_ids is None else page_ids.numel()
    ids_at = None if page_ids is None else _capi.pointer(
        page_ids, torch.int32, (count,), device, "page_ids must be contiguous int32 [n]")
    lengths_at = None if lengths is None else _capi.pointer(
        lengths, torch.int32, (count,), device, "lengths must be contiguous int32, one per page")
    stream = _capi.launch_stream(device)
    if count and pages:
        _capi.call("pg_sparse_key_bounds", codes_at, bounds_at, pages, ids_at, lengths_at, count, heads, stream)


class SelectedPagesDecode(_SegmentDecode):
    """Attention of one token per request over selected INT8 pages, an exact FP16 tail
    and the value center.  ``select`` and ``run`` of one object share its workspace and
    must not overlap on different streams; it belongs to this object alone."""

    def plan(self, indptr, indices: torch.Tensor, last_page_len: torch.Tensor, tail_indptr=None,
             tail_indices: Optional[torch.Tensor] = None, tail_last_page_len: Optional[torch.Tensor] = None,
             *, pages: int, first_pages: int = 1, last_pages: int = 1, num_qo_heads: int = 32,
             num_kv_heads: int = 8, sm_scale: Optional[float] = None, num_cus: Optional[int] = None) -> None:
        """CSR page tables of the history and, with ``tail_indptr``, of the exact pages;
        either may be empty for a request.  Of the history ``pages`` are read for each
        KV head, all of a request that has no more; the first ``first_pages`` and last
        ``last_pages`` of the table are always among them.  ``indices`` and the last
        lengths (device int32) must stay alive until the next ``plan`` and are re-read
        by every call, so captured calls stay valid until the next ``plan``.  Lengths may
        move within [0, 16], and ids may be rewritten in place within the pool; an entry
        below 0 is no page, has no score and is left out.  Waits for the GPU."""
        if pages <= 0:
            raise ValueError("at least one page must be selected")
        if first_pages < 0 or last_pages < 0 or first_pages + last_pages > pages:
            raise ValueError(f"{first_pages} first and {last_pages} last pages do not fit {pages} selected ones")
        host, own_ids = _tables(indptr, indices, last_page_len)
        tail, tail_ids = self._plan_tail(host, tail_indptr, tail_indices, tail_last_page_len)
        tables = (indices, last_page_len, tail_indices, tail_last_page_len)
        _capi.require_current_device(self.workspace, *tables)
        batch = host.numel() - 1
        _capi.call("pg_sparse_plan", host.data_ptr(), _ptr(tail), batch, num_qo_heads, num_kv_heads, pages,
                   first_pages, last_pages, int(num_cus or _num_cus(indices.device)), self.workspace.data_ptr(),
                   self.workspace.numel(), self._plan_ref, _capi.current_stream())
        self._pages = pages
        self._keep_plan(batch, num_qo_heads, num_kv_heads, torch.int8, sm_scale, tables, (own_ids,), tail_ids)

    def _selection(self, selected: torch.Tensor, device: int) -> int:
        return _capi.pointer(selected, torch.int32, (self._batch, self._num_kv_heads, self._pages), device,
                             "selected must be contiguous int32 [B,Hkv,pages]")

    def select(self, q: torch.Tensor, bounds: torch.Tensor, k_page_scale: torch.Tensor,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The pages that ``q`` [B, Hq, 128] (FP16, dense heads) picks: int32
        [B, Hkv, pages], positions in each request's table, ascending, -1 past the last.
        Among equal scores the lowest positions are taken; a query row with an infinity
        or NaN has no say."""
        if not self._planned:
            raise RuntimeError("plan() must be called before select()")
        _check_query(q, self._batch, self._num_qo_heads)
        device = q.get_device()
        if bounds.dim() != 4:
            raise ValueError(_BOUNDS)
        pool = bounds.shape[0]
        bounds_at = _capi.pointer(bounds, torch.int8, (pool, self._num_kv_heads, 2, DIM), device, _BOUNDS)
        _check_scale(k_page_scale, "k_page_scale", pool, self._num_kv_heads)
        if k_page_scale.get_device() != device or self._device != device:
            raise ValueError(_capi.DEVICE_ERROR)
        if pool < self._need:
            self._check_pool(pool, "bounds'")
        out_at = None if out is None else self._selection(out, device)
        stream = _capi.launch_stream(device)
        if out is None:
            out = torch.empty(self._batch, self._num_kv_heads, self._pages, dtype=torch.int32, device=q.device)
            out_at = out.data_ptr()
        _capi.call("pg_sparse_select", self._plan_ref, q.data_ptr(), q.stride(0), bounds_at,
                   k_page_scale.data_ptr(), self._table_ptrs[0], out_at, self.workspace.data_ptr(), stream)
        return out

    def run(self, q: torch.Tensor, kv_cache, k_page_scale: torch.Tensor, v_page_scale: torch.Tensor,
            selected: torch.Tensor, exact_cache=None, value_center: Optional[torch.Tensor] = None,
            sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
            lse: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of ``q`` over the pages at the positions ``selected`` [B, Hkv, pages]
        (``select``'s, or the caller's own: different ones, in any order, those outside
        a table not read; of a request with fewer pages that many entries count).  The rest
        as ``prefix.SharedPrefixDecode.run``."""
        if not self._planned:
            raise RuntimeError("plan() must be called before run()")
        cache_at, exact_at, center_at, out, lse, out_at, lse_at, stream = self._run_args(
            q, kv_cache, k_page_scale, v_page_scale, exact_cache, value_center, out, lse, return_lse)
        selected_at = self._selection(selected, q.get_device())
        indices, last, tail_indices, tail_last = self._table_ptrs
        _capi.call("pg_sparse_run", self._plan_ref, q.data_ptr(), q.stride(0), *cache_at, indices, last, selected_at,
                   *exact_at, tail_indices, tail_last, center_at, out_at, lse_at,
                   float(self._sm_scale if sm_scale is None else sm_scale), self.workspace.data_ptr(), stream)
        return (out, lse) if return_lse else out
