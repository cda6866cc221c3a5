"""The KV cache held in 4 bits: writers, reader-back and attention.

Beside the INT8 pages of ``update`` and ``decode``, the same page tables, exact
FP16 pages and centers over pages of half the bytes.  A page of 16 tokens holds
per KV head one code in [-7, 7] per value and one FP16 scale per token, K and V
apart, of rows centered on the request's channel means:

* ``allocate_pages`` -- the pool: ``codes`` uint8 [pages, Hkv, 2, 1024] and
  ``scales`` FP16 [pages, Hkv, 4, 2, 4] (``include/pagegauge_hip.h`` gives the
  order of the nibbles);
* ``quantize_pages`` -- a prompt's token-major K and V into pages, with the
  centered FP16 copies of its exact pages (the 4-bit ``update.prefill_page_gauge``);
* ``dequantize_pages`` -- back to FP16, for a prompt that continues a cached
  prefix (its attention is the caller's: ``decoder.prefill`` takes whole prompts);
* ``rope_append`` -- one token per request: rotation, centered append to the
  exact pages, and the page that a token completed held in 4 bits (the 4-bit
  ``rope_append_page_gauge_slots``, with ``rotary.RotaryEmbedding``);
* ``Int4PagedDecode`` -- attention of one token per request over 4-bit pages,
  an exact FP16 tail and the value center, planned like
  ``decode.PageGaugeSegmentedDecode``, for 1 to 16 query heads per KV head.

Everything runs on the current stream and nothing but ``plan`` synchronises.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _capi
from .decode import (_check_index, _check_page_ids, _check_query, _host_i32, _host_tables, _num_cus,
                     _page_id_range)
from .rotary import RotaryEmbedding

DIM = 128
PAGE = 16
BLOCK_SHAPE = (2, 1024)
SCALE_SHAPE = (4, 2, 4)

# what the checks below say
_CODES = "4-bit codes must be contiguous uint8 [pages,Hkv,2,1024]"
_SCALES = "4-bit scales must be contiguous float16 [pages,Hkv,4,2,4]"
_CENTERS = "centers must be contiguous float16, [Hkv,128] of each request"
_EXACT_KEY = "exact_key must be contiguous float16 [pages,16,Hkv,128]"
_EXACT_VALUE = "exact_value must be contiguous float16 [pages,16,Hkv,128]"
_PAGE_IDS = "page_ids must be contiguous int32, one per page"
_EXACT_IDS = "exact_page_ids must be contiguous int32, one per page or request"
_CODE_IDS = "code_page_ids must be contiguous int32, one per request"


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def allocate_pages(pages: int, kv_heads: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of a pool, zeroed (every value -8 times a scale of 0)."""
    return (torch.zeros(pages, kv_heads, *BLOCK_SHAPE, device=device, dtype=torch.uint8),
            torch.zeros(pages, kv_heads, *SCALE_SHAPE, device=device, dtype=torch.float16))


def _pool(codes: torch.Tensor, scales: torch.Tensor, heads: int, device: int) -> tuple[int, int, int]:
    """(pages, codes' address, scales' address) of a pool."""
    if codes.dim() != 4:
        raise ValueError(_CODES)
    pages = codes.shape[0]
    return (pages, _capi.pointer(codes, torch.uint8, (pages, heads, 2, 1024), device, _CODES),
            _capi.pointer(scales, torch.float16, (pages, heads, 4, 2, 4), device, _SCALES))


def _ids(ids: Optional[torch.Tensor], count: int, device: int, what: str) -> Optional[int]:
    return None if ids is None else _capi.pointer(ids, torch.int32, (count,), device, what)


def _token_rows(t: torch.Tensor, what: str) -> int:
    """Token stride of FP16 rows [T, H, 128] whose heads are dense."""
    shape = t.shape
    if t.dtype is torch.float16 and len(shape) == 3 and shape[2] == DIM and shape[1] > 0:
        token, head, dim = t.stride()
        if dim == 1 and (head == DIM or shape[1] == 1):
            return token
    raise ValueError(f"{what} must be float16 [T,Hkv,128] rows of dense heads")


def _centers(key_center, value_center, shape: tuple, device: int):
    if key_center is None and value_center is None:
        return None, None
    if key_center is None or value_center is None:
        raise ValueError("key and value centers go together")
    return (_capi.pointer(key_center, torch.float16, shape, device, _CENTERS),
            _capi.pointer(value_center, torch.float16, shape, device, _CENTERS))


def _exact(pages: torch.Tensor, heads: int, device: int, what: str) -> tuple[int, int]:
    """(pages, address) of exact FP16 pages."""
    if pages.dim() != 4:
        raise ValueError(what)
    count = pages.shape[0]
    return count, _capi.pointer(pages, torch.float16, (count, PAGE, heads, DIM), device, what)


def _check_last(indptr: torch.Tensor, last: torch.Tensor, what: str) -> None:
    """The last length of every request with pages lies in [1, 16] (host tensors)."""
    if bool(((indptr[1:] > indptr[:-1]) & ((last < 1) | (last > PAGE))).any()):
        raise ValueError(f"{what} must lie in [1, {PAGE}]")


def quantize_pages(key: torch.Tensor, value: torch.Tensor, codes: torch.Tensor,
                   scales: torch.Tensor, *, page_ids: Optional[torch.Tensor] = None,
                   key_center: Optional[torch.Tensor] = None,
                   value_center: Optional[torch.Tensor] = None,
                   exact_page_ids: Optional[torch.Tensor] = None,
                   exact_key: Optional[torch.Tensor] = None,
                   exact_value: Optional[torch.Tensor] = None) -> None:
    """Hold token-major rows ``key``, ``value`` [T, Hkv, 128] in 4 bits: tokens
    16i .. 16i + 15 in page ``page_ids[i]`` of the pool (device int32
    [ceil(T / 16)]; None: page i), centered on ``key_center``, ``value_center``
    [Hkv, 128] where given.  The rows of a partial last page past T get scale
    0.  With ``exact_page_ids`` those pages are also stored, centered and
    rounded to FP16, in pages ``exact_page_ids[i]`` of ``exact_key`` and
    ``exact_value`` [pages, 16, Hkv, 128].  Ids outside their pool (-1) skip
    the store; the others must differ from each other.  Rows may be strided
    by token, and may not lie in the exact pages."""
    if key.shape != value.shape:
        raise ValueError("token-major K/V must have identical [T,Hkv,128] shapes")
    key_stride, value_stride = _token_rows(key, "K"), _token_rows(value, "V")
    tokens, heads, _ = key.shape
    pages = (tokens + PAGE - 1) // PAGE
    device = key.get_device()
    pool, codes_at, scales_at = _pool(codes, scales, heads, device)
    ids_at = _ids(page_ids, pages, device, _PAGE_IDS)
    exact_ids_at = _ids(exact_page_ids, pages, device, _EXACT_IDS)
    if page_ids is None and pages > pool:
        raise ValueError(f"{pages} pages do not fit a pool of {pool}")
    key_center_at, value_center_at = _centers(key_center, value_center, (heads, DIM), device)
    exact_pages, exact_key_at, exact_value_at = 0, None, None
    if exact_page_ids is not None:
        if exact_key is None or exact_value is None:
            raise ValueError("exact page ids need exact key/value pages")
        exact_pages, exact_key_at = _exact(exact_key, heads, device, _EXACT_KEY)
        count, exact_value_at = _exact(exact_value, heads, device, _EXACT_VALUE)
        exact_pages = min(exact_pages, count)
    if value.get_device() != device:
        raise ValueError(_capi.DEVICE_ERROR)
    stream = _capi.launch_stream(device)
    if tokens == 0 or pool == 0 and exact_pages == 0:
        return
    if pool == 0 or exact_page_ids is not None and exact_pages == 0:
        raise ValueError("a pool without pages holds nothing")
    _capi.call("pg_int4_quantize_pages", key.data_ptr(), key_stride, value.data_ptr(), value_stride,
               key_center_at, value_center_at, codes_at, scales_at, pool, ids_at, exact_ids_at,
               exact_key_at, exact_value_at, exact_pages, tokens, heads, stream)


def dequantize_pages(codes: torch.Tensor, scales: torch.Tensor,
                     page_ids: Optional[torch.Tensor] = None, *, tokens: Optional[int] = None,
                     key_center: Optional[torch.Tensor] = None,
                     value_center: Optional[torch.Tensor] = None,
                     key: Optional[torch.Tensor] = None,
                     value: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(K, V) rows [tokens, Hkv, 128] in FP16 that pages ``page_ids`` (device
    int32; None: the whole pool in order) stand for, ``code * scale + center``.
    ``tokens`` defaults to whole pages.  Ids outside the pool give zeros.
    ``key`` and ``value`` may be given (token rows may be strided).  Scales and
    centers that autograd follows are refused: there is no backward pass."""
    if codes.dim() != 4 or codes.shape[1] == 0:
        raise ValueError(_CODES)
    heads, device = codes.shape[1], codes.get_device()
    pool, codes_at, scales_at = _pool(codes, scales, heads, device)
    pages = pool if page_ids is None else page_ids.numel()
    ids_at = _ids(page_ids, pages, device, _PAGE_IDS)
    tokens = pages * PAGE if tokens is None else int(tokens)
    if not 0 <= tokens <= pages * PAGE:
        raise ValueError(f"{pages} pages hold at most {pages * PAGE} tokens, asked for {tokens}")
    _capi.refuse_gradients(scales, key_center, value_center)
    key_center_at, value_center_at = _centers(key_center, value_center, (heads, DIM), device)
    shape, dense = (tokens, heads, DIM), (heads * DIM, DIM, 1)
    strides = []
    for t in (key, value):
        stride = heads * DIM
        if t is not None:
            if t.shape != shape:
                raise ValueError(f"K and V rows must be [{tokens},{heads},128]")
            stride = _token_rows(t, "K and V")
            if tokens > 1 and stride < heads * DIM:
                raise ValueError("K and V rows must not overlap")
            if t.get_device() != device:
                raise ValueError(_capi.DEVICE_ERROR)
        strides.append(stride)
    stream = _capi.launch_stream(device)
    if key is None:
        key = torch.empty_strided(shape, dense, dtype=torch.float16, device=codes.device)
    if value is None:
        value = torch.empty_strided(shape, dense, dtype=torch.float16, device=codes.device)
    if tokens:
        _capi.call("pg_int4_dequantize_pages", codes_at, scales_at, pool, ids_at, key_center_at,
                   value_center_at, key.data_ptr(), strides[0], value.data_ptr(), strides[1], tokens,
                   heads, stream)
    return key, value


def rope_append(rotary: RotaryEmbedding, query: torch.Tensor, key: torch.Tensor,
                value: torch.Tensor, positions: torch.Tensor, exact_page_ids: torch.Tensor,
                code_page_ids: torch.Tensor, key_center: torch.Tensor, value_center: torch.Tensor,
                rotated_query: torch.Tensor, exact_key: torch.Tensor, exact_value: torch.Tensor,
                codes: torch.Tensor, scales: torch.Tensor) -> None:
    """The cache update of one token per request, in one launch: ``query``
    [B, Hq, 128] and ``key`` [B, Hkv, 128] rotated at ``positions`` (device
    int32 [B]), the query into ``rotated_query``, key and ``value`` minus their
    centers [B, Hkv, 128] into row ``positions % 16`` of page
    ``exact_page_ids[b]`` of ``exact_key`` / ``exact_value``
    [pages, 16, Hkv, 128], and where that is row 15, the completed page in 4
    bits into page ``code_page_ids[b]`` of the pool.

    The tables are ``serving.decode_tables``' or the caller's own.  A request
    with a negative position (padding of a captured batch) is left out whole;
    ids outside their pool skip the store.  The pages of one call must differ
    from each other."""
    if rotary.head_dim != DIM:
        raise ValueError("the cache holds heads of 128 dims")
    query_stride, key_stride = _token_rows(query, "query"), _token_rows(key, "key")
    value_stride = _token_rows(value, "value")
    batch, heads, _ = key.shape
    if value.shape != key.shape or query.shape[0] != batch:
        raise ValueError("query, key and value must have a row per request")
    device = key.get_device()
    positions_at = _ids(positions, batch, device, "positions must be contiguous int32, one per request")
    exact_ids_at = _ids(exact_page_ids, batch, device, _EXACT_IDS)
    code_ids_at = _ids(code_page_ids, batch, device, _CODE_IDS)
    if key_center is None:
        raise ValueError("key and value centers are required")
    key_center_at, value_center_at = _centers(key_center, value_center, (batch, heads, DIM), device)
    rotated_at = _capi.pointer(rotated_query, torch.float16, query.shape, device,
                               "rotated_query must be contiguous float16, shaped like the query")
    exact_pages, exact_key_at = _exact(exact_key, heads, device, _EXACT_KEY)
    count, exact_value_at = _exact(exact_value, heads, device, _EXACT_VALUE)
    pool, codes_at, scales_at = _pool(codes, scales, heads, device)
    if query.get_device() != device or value.get_device() != device \
            or rotary.turns.get_device() != device:
        raise ValueError(_capi.DEVICE_ERROR)
    stream = _capi.launch_stream(device)
    if batch == 0:
        return
    exact_pages = min(exact_pages, count)
    if pool == 0 or exact_pages == 0:
        raise ValueError("a pool without pages holds nothing")
    _capi.call("pg_int4_rope_append", query.data_ptr(), key.data_ptr(), value.data_ptr(), query_stride,
               key_stride, value_stride, positions_at, rotary.turns.data_ptr(), rotary.amplitude,
               rotary.rotary_dim, int(rotary.interleaved), exact_ids_at, code_ids_at, key_center_at,
               value_center_at, rotated_at, exact_key_at, exact_value_at, exact_pages, codes_at,
               scales_at, pool, batch, query.shape[1], heads, stream)


def plan_work_items(indptr, tail_indptr=None, num_qo_heads: int = 32, num_kv_heads: int = 8,
                    num_cus: int = 256):
    """Run the planner on the host only: ``(plan, items [n, 8], item_ptr)``."""
    lib = _capi.library()
    host = _host_i32(indptr)
    tail = None if tail_indptr is None else _host_i32(tail_indptr)
    if host.dim() != 1 or host.numel() < 2 or tail is not None and tail.shape != host.shape:
        raise ValueError("indptr must be a 1-D tensor of batch_size + 1 >= 2 entries")
    batch = host.numel() - 1
    plan = _capi.Int4Plan()
    args = (host.data_ptr(), _ptr(tail), batch, num_qo_heads, num_kv_heads, num_cus,
            ctypes.byref(plan))
    _capi.check(lib.pg_int4_plan_host(*args, None, 0, None), "decode plan")
    items = torch.empty(plan.num_items, 8, dtype=torch.int32)
    item_ptr = torch.empty(batch + 1, dtype=torch.int32)
    _capi.check(lib.pg_int4_plan_host(*args, items.data_ptr(), items.shape[0], item_ptr.data_ptr()),
                "decode plan")
    return plan, items, item_ptr


class Int4PagedDecode:
    """Attention of one token per request over 4-bit history pages, an exact
    FP16 tail and the value center (``plan`` / ``run`` as
    ``decode.PageGaugeSegmentedDecode``).  Runs of one object share its
    workspace and must not overlap on different streams; it belongs to this
    object alone (another one's plan would replace the work list in it)."""

    def __init__(self, workspace: torch.Tensor) -> None:
        if not workspace.is_cuda or workspace.dtype != torch.uint8 or not workspace.is_contiguous() \
                or workspace.data_ptr() % 256:
            raise ValueError("workspace must be a contiguous CUDA uint8 tensor, 256-byte aligned")
        self.workspace = workspace
        self._device = workspace.get_device()
        self._plan = _capi.Int4Plan()
        self._plan_ref = ctypes.byref(self._plan)
        self._planned = False

    def plan(self, indptr, indices: torch.Tensor, last_page_len: torch.Tensor,
             tail_indptr=None, tail_indices: Optional[torch.Tensor] = None,
             tail_last_page_len: Optional[torch.Tensor] = None, num_qo_heads: int = 32,
             num_kv_heads: int = 8, sm_scale: Optional[float] = None,
             num_cus: Optional[int] = None) -> None:
        """CSR page tables of the history and, with ``tail_indptr``, of the
        exact pages; either may be empty for a request.  ``indices`` and the
        last lengths (device int32) must stay alive until the next ``plan``
        and are re-read by every run (lengths within [0, 16] may move), so a
        captured run stays valid until the next ``plan``.  Waits for the GPU."""
        if (tail_indptr is None) != (tail_indices is None) or (tail_indptr is None) != (
                tail_last_page_len is None):
            raise ValueError("tail indptr, indices and last_page_len go together")
        _check_index(indices, "indices")
        _check_index(last_page_len, "last_page_len")
        host, last = _host_tables(indptr, last_page_len, indices)
        _check_last(host, last, "last_page_len")
        tail = tail_range = None
        if tail_indptr is not None:
            _check_index(tail_indices, "tail_indices")
            _check_index(tail_last_page_len, "tail_last_page_len")
            tail, last = _host_tables(tail_indptr, tail_last_page_len, tail_indices, "tail")
            _check_last(tail, last, "tail_last_page_len")
            if tail.numel() != host.numel():
                raise ValueError("history and tail page tables must cover the same batch")
            tail_range = _page_id_range(tail_indices, tail)
        _capi.require_current_device(self.workspace, indices, last_page_len, tail_indices,
                                     tail_last_page_len)
        _capi.call("pg_int4_plan", host.data_ptr(), _ptr(tail), host.numel() - 1, num_qo_heads,
                   num_kv_heads, int(num_cus or _num_cus(indices.device)), self.workspace.data_ptr(),
                   self.workspace.numel(), self._plan_ref, _capi.current_stream())
        self._planned = True
        self._tables = (indices, last_page_len, tail_indices, tail_last_page_len)
        self._table_ptrs = tuple(_ptr(t) for t in self._tables)
        self._id_ranges = (_page_id_range(indices, host), tail_range)
        self._batch = host.numel() - 1
        self._num_qo_heads, self._num_kv_heads = num_qo_heads, num_kv_heads
        self._sm_scale = sm_scale if sm_scale is not None else 1.0 / math.sqrt(DIM)

    @property
    def num_work_items(self) -> int:
        return int(self._plan.num_items)

    def run(self, q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, exact_cache=None,
            value_center: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
            out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
            return_lse: bool = False):
        """Attention of ``q`` [B, Hq, 128] (FP16, dense heads): ``out`` FP16
        [B, Hq, 128], with ``return_lse`` also the base-2 lse float32 [B, Hq].
        ``exact_cache`` is the (K, V) pages of the tail, ``value_center``
        [B, Hkv, 128].  A request without tokens gives its center (or zeros)
        and an lse of -inf.  Queries, pages and centers that autograd follows are
        refused: there is no backward pass."""
        if not self._planned:
            raise RuntimeError("plan() must be called before run()")
        hkv, hq, batch = self._num_kv_heads, self._num_qo_heads, self._batch
        _check_query(q, batch, hq)
        _capi.refuse_gradients(q, value_center)
        device = q.get_device()
        pool, codes_at, scales_at = _pool(codes, scales, hkv, device)
        exact_k_at = exact_v_at = center_at = lse_at = None
        if self._tables[2] is not None:
            if exact_cache is None:
                raise ValueError("a plan with a tail needs the exact pages")
            exact_k, exact_v = exact_cache
            _capi.refuse_gradients(exact_k, exact_v)
            pages, exact_k_at = _exact(exact_k, hkv, device, _EXACT_KEY)
            count, exact_v_at = _exact(exact_v, hkv, device, _EXACT_VALUE)
            if self._id_ranges[1] is not None:
                _check_page_ids(self._id_ranges[1], min(pages, count), "exact tail")
        if self._id_ranges[0] is not None:
            _check_page_ids(self._id_ranges[0], pool, "4-bit")
        if value_center is not None:
            center_at = _capi.pointer(value_center, torch.float16, (batch, hkv, DIM), device, _CENTERS)
        if out is None:
            out = torch.empty_like(q)
            if not out.is_contiguous():
                out = torch.empty(q.shape, device=q.device, dtype=torch.float16)
            out_at = out.data_ptr()
        else:
            out_at = _capi.pointer(out, torch.float16, q.shape, device,
                                   "out must be contiguous float16, shaped like q")
        if lse is not None:
            lse_at = _capi.pointer(lse, torch.float32, (batch, hq), device,
                                   "lse must be contiguous float32 [B,Hq]")
        elif return_lse:
            lse = torch.empty_strided((batch, hq), (hq, 1), dtype=torch.float32, device=q.device)
            lse_at = lse.data_ptr()
        if self._device != device:
            raise ValueError(_capi.DEVICE_ERROR)
        stream = _capi.launch_stream(device)
        indices, last, tail_indices, tail_last = self._table_ptrs
        _capi.call("pg_int4_decode_run", self._plan_ref, q.data_ptr(), q.stride(0), codes_at, scales_at,
                   indices, last, exact_k_at, exact_v_at, tail_indices, tail_last, center_at, hkv * DIM,
                   out_at, lse_at, float(self._sm_scale if sm_scale is None else sm_scale),
                   self.workspace.data_ptr(), stream)
        return (out, lse) if return_lse else out
