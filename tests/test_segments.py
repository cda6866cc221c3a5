"""Attention over shared prefixes and selected pages on the CPU: the planner, and what
is refused before anything reaches the GPU."""

from __future__ import annotations

import ctypes
import random
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from pagegauge_amd import _capi, pages, prefix, sparse

ROOT = Path(__file__).resolve().parents[1]
FIELDS = ("request", "row_first", "rows", "segment", "page_begin", "page_end", "last_page", "tail_begin",
          "tail_end", "last_tail", "slot_at", "split", "table_begin", "table_pages", "block_rows", "reserved")


def _check_plan(segments, own, tail, hq, hkv, cus, kind=torch.int8, selected=0):
    """Every (row, page) that a request sees is read once, into a slot of its own."""
    group = hq // hkv
    indptr = np.concatenate(([3], 3 + np.cumsum(own))).astype(int)
    tail_indptr = None if tail is None else np.concatenate(([1], 1 + np.cumsum(tail))).astype(int)
    shared = np.concatenate(([2], 2 + np.cumsum([s[2] for s in segments]))).astype(int)
    plan, items, slot_ptr, slot_base = prefix.plan_work_items(
        indptr.tolist(), None if tail is None else tail_indptr.tolist(), [s[:2] for s in segments], shared.tolist(),
        hq, hkv, kind, selected, cus)
    items = [dict(zip(FIELDS, row)) for row in items.tolist()]
    slot_ptr, slot_base = slot_ptr.tolist(), slot_base.tolist()
    seen = {}                                    # (request, head, segment or None, "page" / "tail") -> ranges
    used, slots_of = set(), {}
    for it in items:
        most = 256 if it["block_rows"] <= 16 else 512       # page ids of a wave's lanes, or in LDS
        assert it["block_rows"] in (8, 16, 64, 128) and 0 < it["rows"] <= it["block_rows"]
        assert it["page_end"] - it["page_begin"] <= most and it["tail_end"] - it["tail_begin"] <= 256
        if it["block_rows"] > 16:
            assert it["segment"] >= 0 and it["page_begin"] < it["page_end"] and it["slot_at"] >= 0
        parts = 2 if it["block_rows"] == 64 else 1
        for row in range(it["row_first"], it["row_first"] + it["rows"]):
            request, head = it["request"] + row // group, row % group
            s = it["segment"]
            if s >= 0:
                first, end, _ = segments[s]
                assert first == it["request"] and request < end and it["last_page"] == shared[s + 1] - 1
                assert it["tail_begin"] == it["tail_end"]
            else:
                assert row < group
                begin, count = (indptr[request], own[request]) if not selected else (0, min(selected, own[request]))
                assert it["last_page"] == begin + count - 1
                assert (it["table_begin"], it["table_pages"]) == (indptr[request], own[request])
                seen.setdefault((request, head, s, "tail"), []).append((it["tail_begin"], it["tail_end"]))
            seen.setdefault((request, head, s, "page"), []).append((it["page_begin"], it["page_end"]))
            if it["slot_at"] < 0:
                assert slot_ptr[request] == slot_ptr[request + 1]
                slots = [None]
            else:
                slot = slot_base[it["slot_at"] + row // group] + it["split"]
                slots = list(range(slot, slot + parts))
                assert slot_ptr[request] <= slot and slots[-1] < slot_ptr[request + 1]
            assert not used & {(request, head, slot) for slot in slots}
            used |= {(request, head, slot) for slot in slots}
            slots_of.setdefault((request, head), []).extend(slots)
    for r in range(len(own)):
        for h in range(group):
            parts = [(s, "page", shared[s], shared[s + 1]) for s, (a, b, _) in enumerate(segments) if a <= r < b]
            begin = 0 if selected else indptr[r]
            parts.append((-1, "page", begin, begin + (min(selected, own[r]) if selected else own[r])))
            if tail is not None:
                parts.append((-1, "tail", tail_indptr[r], tail_indptr[r + 1]))
            for s, what, lo, hi in parts:
                ranges = sorted(x for x in seen.get((r, h, s, what), []) if x[0] < x[1])
                edges = [lo] + [b for _, b in ranges]
                assert [a for a, _ in ranges] == edges[:-1] and edges[-1] == hi, (r, s, what)
            slots = slots_of[r, h]
            if slots == [None]:
                continue
            assert sorted(slots) == list(range(slot_ptr[r], slot_ptr[r + 1])) and slots
    assert plan.num_items == len(items) and plan.max_slots == max(np.diff(slot_ptr))
    assert plan.partial_rows == slot_ptr[-1]
    assert plan.workspace_bytes >= plan.partial_offset + slot_ptr[-1] * hq * 130 * 4
    return items


@pytest.mark.parametrize("segments,own,tail", [
    ([], [0], None), ([], [1], [0]), ([], [257, 0, 5000], [16, 0, 700]), ([(0, 1, 1)], [0], [0]),
    ([(0, 3, 100)], [0, 4, 0], [0, 1, 0]), ([(0, 256, 1024)], [30] * 256, [16] * 256),
    ([(1, 4, 70), (0, 5, 9), (2, 2, 8), (3, 5, 0), (2, 5, 4000)], [0, 1, 0, 300, 0], [0, 0, 17, 600, 0])])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (16, 1), (7, 1), (64, 16)])
def test_plan_reads_every_page_once(segments, own, tail, hq, hkv):
    for cus in (1, 256):
        for kind in (torch.int8, torch.float16):
            _check_plan(segments, own, tail, hq, hkv, cus, kind)


def test_plans_of_drawn_batches():
    rng = random.Random(11)
    for _ in range(60):
        n = rng.randint(1, 40)
        own = [rng.choice([0, 1, rng.randint(0, 30), rng.randint(0, 900)]) for _ in range(n)]
        tail = [rng.choice([0, 1, 16, rng.randint(0, 300)]) for _ in range(n)]
        segments = [(*sorted((rng.randint(0, n), rng.randint(0, n))), rng.choice([0, 1, rng.randint(0, 2000)]))
                    for _ in range(rng.randint(0, 5))]
        hkv = rng.choice([1, 2, 5, 8])
        hq, cus = hkv * rng.randint(1, 16), rng.choice([1, 100, 256, 304])
        _check_plan(segments, own, tail, hq, hkv, cus)
        _check_plan([], own, tail, hq, hkv, cus, selected=rng.choice([1, 16, 300]))


@pytest.mark.parametrize("args,message", [
    (dict(indptr=[0, 4], num_qo_heads=30), "multiple of KV heads"),
    (dict(indptr=[0, 4], num_qo_heads=17, num_kv_heads=1), "at most 16 query heads"),
    (dict(indptr=[0, 4], num_qo_heads=1025, num_kv_heads=1025), "at most 1024 KV heads"),
    (dict(indptr=[0, 4], num_kv_heads=0), "positive multiple"),
    (dict(indptr=[4, 0]), "non-decreasing"), (dict(indptr=[-1, 4]), "nonnegative"),
    (dict(indptr=[0, 4], tail_indptr=[0, -1]), "nonnegative"),
    (dict(indptr=[0, 4], prefix_requests=[(0, 1)], prefix_indptr=[5, 4]), "non-decreasing"),
    (dict(indptr=[0, 4], prefix_requests=[(0, 2)], prefix_indptr=[0, 4]), "range of the batch"),
    (dict(indptr=[0, 4], prefix_requests=[(1, 0)], prefix_indptr=[0, 4]), "range of the batch"),
    (dict(indptr=[0, 4], prefix_requests=[(-1, 1)], prefix_indptr=[0, 4]), "range of the batch"),
    (dict(indptr=[0, 2 ** 31 - 1]), "too many pages"),
])
def test_plan_refuses(args, message):
    with pytest.raises(RuntimeError, match=message):
        prefix.plan_work_items(**args)


@pytest.mark.parametrize("args", [dict(indptr=[0]), dict(indptr=[0, 4], tail_indptr=[0, 4, 8]),
                                  dict(indptr=[0, 4], prefix_requests=[(0, 1)]),
                                  dict(indptr=[0, 4], kv_data_type=torch.bfloat16),
                                  dict(indptr=[0, 4], prefix_requests=torch.zeros(2, 3))])
def test_plan_refuses_shapes(args):
    with pytest.raises(ValueError):
        prefix.plan_work_items(**args)


def test_item_buffers_are_checked():
    lib = _capi.library()
    plan = _capi.SegmentPlan()
    indptr = torch.tensor([0, 400], dtype=torch.int32)
    items = torch.empty(1, 16, dtype=torch.int32)
    args = (None, None, 0, indptr.data_ptr(), None, 1, 32, 8, _capi.PG_KV_INT8, 0, 256, ctypes.byref(plan))
    assert lib.pg_segment_plan_host(*args, items.data_ptr(), 1, None, None, 0) != 0
    assert "too small" in _capi.last_error()
    assert lib.pg_segment_plan_host(*args, None, 0, None, items.data_ptr(), 0) != 0
    assert "slot buffer too small" in _capi.last_error()
    bad_kind = (*args[:8], 7, *args[9:])
    assert lib.pg_segment_plan_host(*bad_kind, None, 0, None, None, 0) != 0
    assert "INT8 or FP16" in _capi.last_error()


@pytest.mark.parametrize("struct,name", [(_capi.SegmentPlan, "pg_segment_plan"), (_capi.PagePlane, "pg_page_plane")])
def test_structs_mirror_the_header(struct, name):
    text = (ROOT / "include" / "pagegauge_hip.h").read_text()
    body = re.search(rf"typedef struct {name} {{(.*?)}} {name}_t;", text, flags=re.S).group(1)
    fields = re.findall(r"(int32_t|int64_t|void\*)\s+(\w+);", body)
    types = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "void*": ctypes.c_void_p}
    assert [(n, types[t]) for t, n in fields] == list(struct._fields_)


def test_c_entries_refuse_before_a_launch():
    """Arguments that no launch may see; every pointer here is the host's and is not read."""
    lib = _capi.library()
    ints = torch.zeros(64, dtype=torch.int32)
    at = ints.data_ptr() + (-ints.data_ptr()) % 16
    plane = (_capi.PagePlane * 1)(_capi.PagePlane(at, 16, 16, 1, 0))
    bad_plane = (_capi.PagePlane * 1)(_capi.PagePlane(at, 16, 8, 1, 0))
    plan = _capi.SegmentPlan()
    for call, message in (
            (lambda: lib.pg_copy_pages(None, 1, 4, at, at, 1, None), "null planes"),
            (lambda: lib.pg_copy_pages(plane, 1, 2 ** 31, at, at, 1, None), "2\\^31"),
            (lambda: lib.pg_copy_pages(plane, 1, 4, None, at, 1, None), "null page ids"),
            (lambda: lib.pg_copy_pages(bad_plane, 1, 4, at, at, 1, None), "overlap"),
            (lambda: lib.pg_pool_adjust(at + 4, 4, at, 1, 1, None), "aligned"),
            (lambda: lib.pg_pool_adjust(None, 4, at, 1, 1, None), "null pool"),
            (lambda: lib.pg_pool_take(at, 4, at, -1, None), "nonnegative"),
            (lambda: lib.pg_pool_stage_compaction(at, 4, None, at, at, at, None), "null output"),
            (lambda: lib.pg_pool_commit_compaction(at, 4, at, at, 5, None), "more moves"),
            (lambda: lib.pg_rewrite_ids(at, None, 4, 4, at, None), "null page ids"),
            (lambda: lib.pg_sparse_key_bounds(at, at + 4, 4, None, None, 4, 8, None), "aligned"),
            (lambda: lib.pg_sparse_key_bounds(at, at, 4, None, None, 5, 8, None), "more pages"),
            (lambda: lib.pg_sparse_key_bounds(at, at, 4, None, None, 4, 0, None), "KV heads"),
            (lambda: lib.pg_sparse_plan(at, None, 1, 32, 8, 0, 0, 0, 256, at, 1 << 20, ctypes.byref(plan), None), "at least one"),
            (lambda: lib.pg_sparse_plan(at, None, 1, 32, 8, 4, 3, 2, 256, at, 1 << 20, ctypes.byref(plan), None), "fit the selection"),
            (lambda: lib.pg_sparse_plan(at, None, 65536, 32, 8, 4, 1, 1, 256, at, 1 << 20, ctypes.byref(plan), None), "65535"),
            (lambda: lib.pg_sparse_select(ctypes.byref(plan), at, 128, at, at, at, at, at, None), "not one of pg_sparse_plan"),
            (lambda: lib.pg_prefix_run(ctypes.byref(plan), at, 128, *[at] * 14, None, 0.1, at, None), "not one of"),
            (lambda: lib.pg_prefix_run(ctypes.byref(plan), at, 128, *[at] * 14, None, 0.0, at, None), "sm_scale"),
            (lambda: lib.pg_prefix_run(None, at, 128, *[at] * 14, None, 0.1, at, None), "null run"),
            (lambda: lib.pg_sparse_run(ctypes.byref(plan), at + 4, 128, *[at] * 13, None, 0.1, at, None), "aligned")):
        assert call() != 0, message
        assert re.search(message, _capi.last_error()), (message, _capi.last_error())


def test_cpu_tensors_are_refused():
    plane, ids = torch.zeros(4, 8), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: pages.copy_pages([plane], ids, ids), lambda: pages.rewrite_ids(ids, ids),
                 lambda: pages.PagePool(4, device="cpu").take(1), lambda: pages.PagePool(4, device="cpu").share(ids),
                 lambda: pages.PagePool(4, device="cpu").stage_compaction(),
                 lambda: sparse.key_bounds(torch.zeros(4, 16, 2, 128, dtype=torch.int8),
                                           sparse.allocate_bounds(4, 2, "cpu")),
                 lambda: prefix.SharedPrefixDecode(torch.empty(1024, dtype=torch.uint8)),
                 lambda: sparse.SelectedPagesDecode(torch.empty(1024, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            call()


def test_page_ids_are_looked_at_again_before_they_are_refused(monkeypatch):
    """A table rewritten in place after the plan; entries below 0 are no pages."""
    from pagegauge_amd import decode

    monkeypatch.setattr(decode, "CHECK_PAGE_IDS", True)
    ids = torch.tensor([9, 3, 7, 12], dtype=torch.int32)
    planned = prefix._PageIds(ids, torch.tensor([1, 4], dtype=torch.int32))
    planned.check(13, "KV")
    with pytest.raises(ValueError, match=r"KV page ids span \[3, 12\] but the pool holds 12 pages"):
        planned.check(12, "KV")
    ids.copy_(torch.tensor([99, 2, -1, 5]))
    planned.check(6, "KV")
    with pytest.raises(ValueError, match=r"span \[0, 5\]"):
        planned.check(5, "KV")
    ids.fill_(-1)                                # page 0 is read in their place
    planned.check(1, "KV")
    monkeypatch.setattr(decode, "CHECK_PAGE_IDS", False)
    for unchecked in (planned, prefix._PageIds(ids, torch.tensor([1, 4], dtype=torch.int32))):
        with pytest.raises(ValueError, match="no pages"):
            unchecked.check(0, "KV")
    empty = prefix._PageIds(ids, torch.tensor([0, 0], dtype=torch.int32))
    empty.check(0, "KV")
