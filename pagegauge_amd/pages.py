"""Pages of a pool that requests share: counted, handed out, copied, moved together.

The pools of the other modules (INT8 codes and scales, 4-bit codes and scales, exact
FP16 pages) are planes that share page ids: page p of a request's table is page p
of each of them.  Here

* ``PagePool`` -- the users of each page: a request that forks shares its parent's
  pages (``share``), takes fresh ones for what it will write (``take``), and gives
  all of them back (``release``);
* ``copy_pages`` -- pages copied in any number of planes in one launch: a child's own
  copy of the exact pages, or of the page that it goes on writing;
* ``PagePool.stage_compaction``, ``rewrite_ids``, ``PagePool.commit_compaction`` -- the
  fewest moves that bring the pages in use to the front of the pool, the page
  tables after them, and the counts.

Results do not depend on the order in which the GPU works: pages are handed out and
moved in the order of their ids.  Everything runs on the current stream, nothing
synchronises, and every call can be captured (with ``out`` where it gives ids).
Calls that change a pool or its pages must follow each other on one stream.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional, Sequence

import torch

from . import _capi

NO_PAGE = -1


def _ids(ids: torch.Tensor, device: int, what: str) -> int:
    if ids.dim() != 1:
        raise ValueError(f"{what} must be contiguous int32 [n]")
    return _capi.pointer(ids, torch.int32, ids.shape, device, f"{what} must be contiguous int32 [n]")


@functools.lru_cache(maxsize=1024)
def _plane(shape: tuple, strides: tuple, size: int, page_dim: int) -> tuple[int, tuple]:
    """(pages, (page bytes, page stride, rows, row stride), in bytes) of a plane."""
    if len(shape) <= page_dim:
        raise ValueError(f"planes must have their pages in dimension {page_dim}")
    dense = 1
    for extent, stride in zip(reversed(shape[page_dim + 1:]), reversed(strides[page_dim + 1:])):
        if extent != 1 and stride != dense:
            raise ValueError("each page of a plane must be contiguous")
        dense *= extent
    pages, rows = shape[page_dim], shape[0] if page_dim else 1
    page_bytes, page_stride = dense * size, strides[page_dim] * size
    row_stride = strides[0] * size if page_dim else 0
    if pages <= 1:
        page_stride = max(page_stride, page_bytes)
    by_rows = row_stride >= (pages - 1) * page_stride + page_bytes
    by_pages = row_stride >= page_bytes and page_stride >= (rows - 1) * row_stride + page_bytes
    if page_stride < page_bytes or (rows > 1 and not by_rows and not by_pages):
        raise ValueError("pages of a plane must not overlap")
    return pages, (page_bytes, page_stride, rows, row_stride)


def copy_pages(planes: Sequence[torch.Tensor], source: torch.Tensor, target: torch.Tensor, *,
               page_dim: int = 0) -> None:
    """Copy page ``source[i]`` to page ``target[i]`` (device int32 [n]) in every plane:
    tensors of any type with their pages in dimension ``page_dim``, 0, or 1 for
    layers of a pool [layers, pages, ...]; each page contiguous.  Ids outside the
    pool (-1) skip their copy.  Targets must differ from each other and be no sources
    of the same call; a source may go to several targets."""
    if page_dim not in (0, 1):
        raise ValueError("page_dim must be 0 or 1")
    if source.shape != target.shape:
        raise ValueError("source and target must have one id per copy")
    if isinstance(planes, torch.Tensor):
        raise ValueError("planes must be a sequence of tensors")
    planes = tuple(planes)
    if not planes:
        raise ValueError("no planes to copy")
    _capi.refuse_gradients(*planes)
    device, pages = source.get_device(), None
    source_at, target_at = _ids(source, device, "source"), _ids(target, device, "target")
    entries = []                                    # pg_page_plane_t: five 64-bit fields
    for plane in planes:
        if plane.get_device() != device:
            raise ValueError(_capi.DEVICE_ERROR)
        here, place = _plane(plane.shape, plane.stride(), plane.element_size(), page_dim)
        if pages is None:
            pages = here
        if here != pages:
            raise ValueError("planes must have the same number of pages")
        if place[0] and place[2] and pages:
            entries += (plane.data_ptr(), *place)
    stream = _capi.launch_stream(device)
    moves = source.shape[0]
    if entries and moves:
        _capi.call("pg_copy_pages", (ctypes.c_int64 * len(entries))(*entries), len(entries) // 5, pages, source_at,
                   target_at, moves, stream)


def rewrite_ids(ids: torch.Tensor, remap: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``remap[ids[i]]`` for a table of page ids (device int32, any shape); ids outside
    ``remap`` stay as they are.  ``out`` may be ``ids``.  The entry of a page without
    users becomes -1: calls of ``prefix`` and ``sparse`` planned over the table leave it
    out, those of ``decode`` and ``int4`` take ids of the pool alone, so a request that
    has ended leaves their tables first."""
    device = ids.get_device()
    what = "ids and out must be contiguous int32, shaped alike"
    ids_at = _capi.pointer(ids, torch.int32, ids.shape, device, what)
    remap_at = _ids(remap, device, "remap")
    out_at = None if out is None else _capi.pointer(out, torch.int32, ids.shape, device, what)
    stream = _capi.launch_stream(device)
    if out is None:
        out = torch.empty_like(ids)
        out_at = out.data_ptr()
    if ids.numel():
        _capi.call("pg_rewrite_ids", ids_at, remap_at, remap.numel(), ids.numel(), out_at, stream)
    return out


class Moves(NamedTuple):
    """A staged compaction, device int32: page ``source[i]`` goes to page ``target[i]``
    (-1 past the last move), page p of a table is page ``remap[p]`` afterwards (-1: it was
    free), and the first ``live[0]`` pages of the pool are then those in use."""

    source: torch.Tensor
    target: torch.Tensor
    remap: torch.Tensor
    live: torch.Tensor


class PagePool:
    """Users per page of a pool: ``refs`` (device int32 [pages], zero: free), which may
    be read, or written in place, like any tensor."""

    def __init__(self, pages: int, device="cuda") -> None:
        if not 0 <= pages < 2 ** 31:
            raise ValueError("a pool holds 0 to 2^31 - 1 pages")
        self._refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self._device = self._refs.get_device()

    @property
    def refs(self) -> torch.Tensor:
        return self._refs

    @property
    def pages(self) -> int:
        return self._refs.shape[0]

    def _adjust(self, ids: torch.Tensor, by: int) -> None:
        ids_at = _ids(ids, self._device, "page ids")
        stream = _capi.launch_stream(self._device)
        if ids.numel():
            _capi.call("pg_pool_adjust", self._refs.data_ptr(), self.pages, ids_at, ids.numel(), by, stream)

    def share(self, ids: torch.Tensor, users: int = 1) -> None:
        """``users`` more users of each of the pages ``ids`` (device int32 [n]).  Ids may
        repeat; those outside the pool (-1) are skipped.  A count that reaches 2^31 - 1 stays
        there: the page is never free again, but by a write to ``refs``."""
        if not 0 < users < 2 ** 31:
            raise ValueError("users must be positive")
        self._adjust(ids, users)

    def release(self, ids: torch.Tensor, users: int = 1) -> None:
        """``users`` fewer users of each of the pages, not below none; a count of 2^31 - 1
        stays."""
        if not 0 < users < 2 ** 31:
            raise ValueError("users must be positive")
        self._adjust(ids, -users)

    def take(self, count: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The ``count`` lowest free pages, ascending (device int32 [count], -1 past
        the last free one); each has one user then."""
        if count < 0:
            raise ValueError("the count must be nonnegative")
        out_at = None if out is None else _capi.pointer(out, torch.int32, (count,), self._device,
                                                        "out must be contiguous int32 [count]")
        stream = _capi.launch_stream(self._device)
        if out is None:
            out = torch.empty(count, dtype=torch.int32, device=self._refs.device)
            out_at = out.data_ptr()
        if count:
            _capi.call("pg_pool_take", self._refs.data_ptr(), self.pages, out_at, count, stream)
        return out

    def stage_compaction(self, out: Optional[Moves] = None) -> Moves:
        """The moves that bring the pages in use to the front of the pool.  Nothing has
        moved yet: ``copy_pages(planes, moves.source, moves.target)`` for the pages,
        ``rewrite_ids(table, moves.remap)`` for every table, ``commit_compaction(moves)``
        for the counts, on the same stream, before anything else changes the pool.
        ``out`` may hold an earlier call's tensors."""
        pages, device = self.pages, self._device
        half = pages // 2
        what = "out must be the tensors of a compaction of this pool"
        stream = _capi.launch_stream(device)
        if out is None:
            # one allocation, remap (16-byte aligned) in front
            whole = torch.empty(pages + 2 * half + 1, dtype=torch.int32, device=self._refs.device)
            remap, source, target, live = whole.split_with_sizes((pages, half, half, 1))
            out = Moves(source, target, remap, live)
            remap_at = whole.data_ptr()
            source_at = remap_at + 4 * pages
            at = source_at, source_at + 4 * half, remap_at, source_at + 8 * half
        else:
            at = [_capi.pointer(t, torch.int32, (n,), device, what) for t, n in zip(out, (half, half, pages, 1))]
        _capi.call("pg_pool_stage_compaction", self._refs.data_ptr(), pages, *at, stream)
        return out

    def commit_compaction(self, moves: Moves) -> None:
        """Move the counts along, once the pages have been copied."""
        source_at = _ids(moves.source, self._device, "source")
        target_at = _capi.pointer(moves.target, torch.int32, moves.source.shape, self._device,
                                  "source and target must have one id per move")
        stream = _capi.launch_stream(self._device)
        if moves.source.numel():
            _capi.call("pg_pool_commit_compaction", self._refs.data_ptr(), self.pages, source_at, target_at,
                       moves.source.numel(), stream)
