"""Attention of single tokens where requests share the beginnings of their contexts.

Requests that fork from one prompt, or that follow one long document or
instruction, hold the same pages at the front of their tables.
``SharedPrefixDecode`` reads each shared page once for all of them: the prefix's
keys and values meet the query rows of every request that has it in one product,
and the partial softmax states join with those of a request's own pages and its
exact FP16 tail.  Prefixes may nest (a common instruction, then a document, then
the forks of one answer).

Pages are INT8 (``decode.PageGaugeSegmentedDecode``'s: codes, and a scale per page
and KV head) or FP16 (``decode.BatchDecodeWithPagedKVCacheWrapper``'s), with 1 to
16 query heads per KV head.  Keys that one request sees must be centered alike:
requests keep the key center of the prompt that they share (forks do).  The value
center is one too: codes of shared values hold what that center left.

Everything runs on the current stream and nothing but ``plan`` synchronises.  (Where page
ids are checked, as ``decode.CHECK_PAGE_IDS`` says, a call with fewer pages than the ids
asked for when last looked at looks again, which does too.)
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _capi
from .decode import (_check_index, _check_page_ids, _check_query, _host_i32, _host_tables, _num_cus,
                     _page_id_range)

DIM = 128
PAGE = 16

_KINDS = {torch.int8: _capi.PG_KV_INT8, torch.float16: _capi.PG_KV_FP16}

# what the checks below say
_CENTERS = "centers must be contiguous float16 [B,Hkv,128]"
_CACHE = {dtype: f"k_cache and v_cache must be contiguous {name} [pages,16,Hkv,128], as planned"
          for dtype, name in ((torch.int8, "int8"), (torch.float16, "float16"))}
_SCALES = "k_page_scale and v_page_scale must be contiguous float16 [pages,Hkv]"
_EXACT = "exact_key and exact_value must be contiguous float16 [pages,16,Hkv,128]"


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _check_last(indptr: torch.Tensor, last: torch.Tensor, what: str) -> None:
    """The last length of every table with pages lies in [1, 16] (host tensors)."""
    if bool(((indptr[1:] > indptr[:-1]) & ((last < 1) | (last > PAGE))).any()):
        raise ValueError(f"{what} must lie in [1, {PAGE}]")


class _PageIds:
    """The page ids of a planned table, and (where ``decode.CHECK_PAGE_IDS`` is set) between
    which they lay when last looked at."""

    def __init__(self, indices: torch.Tensor, host_indptr: torch.Tensor) -> None:
        self._indices, self._indptr = indices, host_indptr
        self._empty = int(host_indptr[0]) == int(host_indptr[-1])
        self._look()

    def _look(self) -> None:
        found = _page_id_range(self._indices, self._indptr)
        self._range = None if found is None else tuple(max(i, 0) for i in found)

    @property
    def need(self) -> int:
        """The fewest pages of a pool that ``check`` takes without another look."""
        return 0 if self._empty else 1 if self._range is None else self._range[1] + 1

    def check(self, pool_pages: int, what: str) -> None:
        """All ids are of a pool of so many pages.  Tables may be rewritten in place after the
        plan: one whose ids were too large is looked at again before it is refused, which waits
        for the GPU and so is left out while a graph is captured."""
        # in the place of an entry below 0, which is no page, the first one is read
        if pool_pages == 0 and not self._empty:
            raise ValueError(f"{what} page tables with entries, but the pool holds no pages")
        if self._range is None or self._range[1] < pool_pages:
            return
        if not (self._indices.is_cuda and torch.cuda.is_current_stream_capturing()):
            self._look()
        _check_page_ids(self._range, pool_pages, what)


def _tables(indptr, indices, last, what: str = ""):
    """Host indptr of a checked CSR page table, and its page ids."""
    name = f"{what}_" if what else ""
    _check_index(indices, f"{name}indices")
    _check_index(last, f"{name}last_page_len")
    host, host_last = _host_tables(indptr, last, indices, what)
    _check_last(host, host_last, f"{name}last_page_len")
    return host, _PageIds(indices, host)


def _prefix_ranges(prefix_requests) -> torch.Tensor:
    """Host int32 [S, 2] of the prefixes' requests."""
    ranges = prefix_requests if isinstance(prefix_requests, torch.Tensor) else \
        torch.tensor([tuple(r) for r in prefix_requests], dtype=torch.int32).reshape(-1, 2)
    if ranges.dim() != 2 or ranges.shape[1] != 2:
        raise ValueError("prefix_requests must be (first, end) of each prefix's requests, [S, 2]")
    return _host_i32(ranges)


def plan_work_items(indptr, tail_indptr=None, prefix_requests=(), prefix_indptr=(0,), num_qo_heads: int = 32,
                    num_kv_heads: int = 8, kv_data_type=torch.int8, selected_pages: int = 0,
                    num_cus: int = 256):
    """Run the planner on the host only: ``(plan, items [n, 16], slot_ptr [B + 1],
    slot_base)``, as ``pg_segment_plan_host`` gives them."""
    lib = _capi.library()
    host, ranges, shared = _host_i32(indptr), _prefix_ranges(prefix_requests), _host_i32(prefix_indptr)
    tail = None if tail_indptr is None else _host_i32(tail_indptr)
    if host.dim() != 1 or host.numel() < 2 or tail is not None and tail.shape != host.shape:
        raise ValueError("indptr must be a 1-D tensor of batch_size + 1 >= 2 entries")
    if shared.shape != (len(ranges) + 1,):
        raise ValueError("prefix_indptr must have one entry per prefix and one more")
    if kv_data_type not in _KINDS:
        raise ValueError("pages must be int8 or float16")
    batch, plan = host.numel() - 1, _capi.SegmentPlan()
    args = (ranges.data_ptr(), shared.data_ptr(), len(ranges), host.data_ptr(), _ptr(tail), batch, num_qo_heads,
            num_kv_heads, _KINDS[kv_data_type], selected_pages, num_cus, ctypes.byref(plan))
    _capi.check(lib.pg_segment_plan_host(*args, None, 0, None, None, 0), "decode plan")
    items = torch.empty(plan.num_items, 16, dtype=torch.int32)
    slot_ptr = torch.empty(batch + 1, dtype=torch.int32)
    slot_base = torch.empty(plan.slot_base_count, dtype=torch.int32)
    _capi.check(lib.pg_segment_plan_host(*args, items.data_ptr(), items.shape[0], slot_ptr.data_ptr(),
                                         slot_base.data_ptr(), slot_base.numel()), "decode plan")
    return plan, items, slot_ptr, slot_base


class _SegmentDecode:
    """What attention over shared prefixes and over selected pages have in common:
    the workspace with its plan, and the checks of a run."""

    def __init__(self, workspace: torch.Tensor) -> None:
        if not workspace.is_cuda or workspace.dtype != torch.uint8 or not workspace.is_contiguous() \
                or workspace.data_ptr() % 256:
            raise ValueError("workspace must be a contiguous CUDA uint8 tensor, 256-byte aligned")
        self.workspace = workspace
        self._device = workspace.get_device()
        self._plan = _capi.SegmentPlan()
        self._plan_ref = ctypes.byref(self._plan)
        self._planned = False

    @property
    def num_work_items(self) -> int:
        return int(self._plan.num_items)

    @property
    def workspace_bytes(self) -> int:
        """Bytes of the workspace that the plan uses."""
        return int(self._plan.workspace_bytes)

    def _plan_tail(self, host, tail_indptr, tail_indices, tail_last_page_len):
        if (tail_indptr is None) != (tail_indices is None) or (tail_indptr is None) != (
                tail_last_page_len is None):
            raise ValueError("tail indptr, indices and last_page_len go together")
        if tail_indptr is None:
            return None, None
        tail, tail_ids = _tables(tail_indptr, tail_indices, tail_last_page_len, "tail")
        if tail.numel() != host.numel():
            raise ValueError("history and tail page tables must cover the same batch")
        return tail, tail_ids

    def _keep_plan(self, batch, num_qo_heads, num_kv_heads, kv_data_type, sm_scale, tables, page_ids, tail_ids):
        self._planned = True
        self._batch, self._num_qo_heads, self._num_kv_heads = batch, num_qo_heads, num_kv_heads
        self._kv_dtype = kv_data_type
        self._sm_scale = sm_scale if sm_scale is not None else 1.0 / math.sqrt(DIM)
        self._tables = tables                       # alive, and where the kernels read
        self._table_ptrs = tuple(_ptr(t) for t in tables)
        self._page_ids, self._tail_ids = page_ids, () if tail_ids is None else (tail_ids,)
        self._need, self._tail_need = (max((ids.need for ids in t), default=0) for t in (page_ids, self._tail_ids))

    def _check_pool(self, pool_pages: int, what: str) -> None:
        """A pool with fewer pages than the tables needed when last looked at."""
        for ids in self._page_ids:
            ids.check(pool_pages, what)
        self._need = max(ids.need for ids in self._page_ids)

    def _check_exact(self, pool_pages: int) -> None:
        for ids in self._tail_ids:
            ids.check(pool_pages, "exact tail")
            self._tail_need = ids.need

    def _run_args(self, q, kv_cache, k_page_scale, v_page_scale, exact_cache, value_center, out, lse, return_lse):
        """Checked pointers of a run, and its outputs."""
        hkv, hq, batch = self._num_kv_heads, self._num_qo_heads, self._batch
        _check_query(q, batch, hq)
        k_cache, v_cache = kv_cache
        device, dtype = q.get_device(), self._kv_dtype
        _capi.refuse_gradients(q, value_center, k_cache, v_cache, k_page_scale, v_page_scale)
        if k_cache.dim() != 4 or v_cache.dim() != 4:
            raise ValueError(_CACHE[dtype])
        k_pages, v_pages = k_cache.shape[0], v_cache.shape[0]
        cache_at = [_capi.pointer(k_cache, dtype, (k_pages, PAGE, hkv, DIM), device, _CACHE[dtype]),
                    _capi.pointer(v_cache, dtype, (v_pages, PAGE, hkv, DIM), device, _CACHE[dtype]), None, None]
        if dtype is torch.int8:
            if k_page_scale is None or v_page_scale is None:
                raise ValueError("INT8 pages need k_page_scale and v_page_scale")
            cache_at[2] = _capi.pointer(k_page_scale, torch.float16, (k_pages, hkv), device, _SCALES)
            cache_at[3] = _capi.pointer(v_page_scale, torch.float16, (v_pages, hkv), device, _SCALES)
        elif k_page_scale is not None or v_page_scale is not None:
            raise ValueError("FP16 pages have no scales")
        if min(k_pages, v_pages) < self._need:
            self._check_pool(min(k_pages, v_pages), "KV")
        exact_at = (None, None)
        if self._tables[-1] is not None:
            if exact_cache is None:
                raise ValueError("a plan with a tail needs the exact pages")
            exact_k, exact_v = exact_cache
            _capi.refuse_gradients(exact_k, exact_v)
            if exact_k.dim() != 4 or exact_v.dim() != 4:
                raise ValueError(_EXACT)
            k_pages, v_pages = exact_k.shape[0], exact_v.shape[0]
            exact_at = (_capi.pointer(exact_k, torch.float16, (k_pages, PAGE, hkv, DIM), device, _EXACT),
                        _capi.pointer(exact_v, torch.float16, (v_pages, PAGE, hkv, DIM), device, _EXACT))
            if min(k_pages, v_pages) < self._tail_need:
                self._check_exact(min(k_pages, v_pages))
        center_at = lse_at = None
        if value_center is not None:
            center_at = _capi.pointer(value_center, torch.float16, (batch, hkv, DIM), device, _CENTERS)
        if out is not None:
            out_at = _capi.pointer(out, torch.float16, q.shape, device,
                                   "out must be contiguous float16, shaped like q")
        if lse is not None:
            lse_at = _capi.pointer(lse, torch.float32, (batch, hq), device,
                                   "lse must be contiguous float32 [B,Hq]")
        if self._device != device:
            raise ValueError(_capi.DEVICE_ERROR)
        stream = _capi.launch_stream(device)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            out_at = out.data_ptr()
        if lse is None and return_lse:
            lse = torch.empty((batch, hq), dtype=torch.float32, device=q.device)
            lse_at = lse.data_ptr()
        return cache_at, exact_at, center_at, out, lse, out_at, lse_at, stream


class SharedPrefixDecode(_SegmentDecode):
    """Attention of one token per request over shared prefixes, a request's own pages,
    an exact FP16 tail and the value center (``plan`` / ``run`` as
    ``decode.PageGaugeSegmentedDecode``).  Runs of one object share its workspace and
    must not overlap on different streams; it belongs to this object alone."""

    def plan(self, prefix_requests, prefix_indptr, prefix_indices: torch.Tensor,
             prefix_last_page_len: torch.Tensor, indptr, indices: torch.Tensor,
             last_page_len: torch.Tensor, tail_indptr=None, tail_indices: Optional[torch.Tensor] = None,
             tail_last_page_len: Optional[torch.Tensor] = None, num_qo_heads: int = 32,
             num_kv_heads: int = 8, sm_scale: Optional[float] = None, kv_data_type=torch.int8,
             num_cus: Optional[int] = None) -> None:
        """``prefix_requests``: (first, end) of the neighbouring requests that have
        each prefix, [S, 2], in any order, nested or overlapping.  CSR page tables of
        the prefixes, of the requests' own pages and, with ``tail_indptr``, of the
        exact pages; any of them may be empty, of a request or as a whole.
        ``indices`` and the last lengths (device int32) must stay alive until the next
        ``plan`` and are re-read by every run, so a captured run stays valid until the
        next ``plan``.  Lengths may move within [0, 16], and ids may be rewritten in
        place within the pool; an entry below 0 is no page and is left out.  Waits for
        the GPU."""
        if kv_data_type not in _KINDS:
            raise ValueError("pages must be int8 or float16")
        ranges = _prefix_ranges(prefix_requests)
        host, own_ids = _tables(indptr, indices, last_page_len)
        tail, tail_ids = self._plan_tail(host, tail_indptr, tail_indices, tail_last_page_len)
        shared, page_ids = _host_i32(prefix_indptr), [own_ids]
        if shared.shape != (len(ranges) + 1,):
            raise ValueError("prefix_indptr must have one entry per prefix and one more")
        if len(ranges):
            shared, shared_ids = _tables(prefix_indptr, prefix_indices, prefix_last_page_len, "prefix")
            page_ids.append(shared_ids)
        else:
            _check_index(prefix_indices, "prefix_indices")
            _check_index(prefix_last_page_len, "prefix_last_page_len")
        tables = (prefix_indices, prefix_last_page_len, indices, last_page_len, tail_indices, tail_last_page_len)
        _capi.require_current_device(self.workspace, *tables)
        batch = host.numel() - 1
        _capi.call("pg_prefix_plan", ranges.data_ptr(), shared.data_ptr(), len(ranges), host.data_ptr(), _ptr(tail),
                   batch, num_qo_heads, num_kv_heads, _KINDS[kv_data_type], int(num_cus or _num_cus(indices.device)),
                   self.workspace.data_ptr(), self.workspace.numel(), self._plan_ref, _capi.current_stream())
        self._keep_plan(batch, num_qo_heads, num_kv_heads, kv_data_type, sm_scale, tables,
                        page_ids, tail_ids)

    def run(self, q: torch.Tensor, kv_cache, k_page_scale: Optional[torch.Tensor] = None,
            v_page_scale: Optional[torch.Tensor] = None, exact_cache=None,
            value_center: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
            out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of ``q`` [B, Hq, 128] (FP16, dense heads): ``out`` FP16 [B, Hq, 128],
        with ``return_lse`` also the base-2 lse float32 [B, Hq].  ``kv_cache`` is the
        (K, V) pages of prefixes and own tables, with INT8 pages their scales
        [pages, Hkv]; ``exact_cache`` the (K, V) pages of the tail, ``value_center``
        [B, Hkv, 128].  A request without tokens gives its center (or zeros) and an lse
        of -inf.  Weights of prefixes with up to 32 query rows (requests times heads of a
        KV head's group), of own pages and of the tail are good to 2^-20 of themselves
        beside their scores' rounding, those of larger prefixes to 2^-11, so that an output
        is off by that part of the weighted mean of |V|.  Tensors that autograd follows are
        refused: there is no backward pass."""
        if not self._planned:
            raise RuntimeError("plan() must be called before run()")
        cache_at, exact_at, center_at, out, lse, out_at, lse_at, stream = self._run_args(
            q, kv_cache, k_page_scale, v_page_scale, exact_cache, value_center, out, lse, return_lse)
        prefix_ids, prefix_last, indices, last, tail_indices, tail_last = self._table_ptrs
        _capi.call("pg_prefix_run", self._plan_ref, q.data_ptr(), q.stride(0), *cache_at, prefix_ids, prefix_last,
                   indices, last, *exact_at, tail_indices, tail_last, center_at, out_at, lse_at,
                   float(self._sm_scale if sm_scale is None else sm_scale), self.workspace.data_ptr(), stream)
        return (out, lse) if return_lse else out
