"""The 4-bit cache on the CPU: the planner, the layout and what is refused."""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest
import torch

from int4_helpers import nibble_maps
from pagegauge_amd import _capi, int4, rotary


def test_every_value_has_one_nibble():
    for where in nibble_maps():
        assert len({tuple(w) for w in where}) == 2048


def _check_plan(pages, tail, hq, hkv, cus):
    indptr = np.concatenate(([3], 3 + np.cumsum(pages)))
    tail_indptr = np.concatenate(([0], np.cumsum(tail)))
    plan, items, item_ptr = int4.plan_work_items(indptr.tolist(), tail_indptr.tolist(), hq, hkv, cus)
    assert plan.num_items == len(items) == item_ptr[-1] and plan.batch_size == len(pages)
    assert bool(plan.has_history) == (sum(pages) > 0)
    most = 0
    for b in range(len(pages)):
        own = items[item_ptr[b]:item_ptr[b + 1]].tolist()
        assert own and all(i[0] == b and i[7] == len(own) for i in own)
        most = max(most, len(own))
        for begin, end, last, (lo, hi) in ((1, 2, 3, indptr[b:b + 2]), (4, 5, 6, tail_indptr[b:b + 2])):
            assert own[0][begin] == lo and own[-1][end] == hi
            assert all(x[end] == y[begin] for x, y in zip(own, own[1:]))
            assert all(x[begin] <= x[end] and x[last] == hi - 1 for x in own)
        assert all(i[2] - i[1] <= 256 for i in own)       # page ids a wave's lanes can hold
    assert plan.max_items_per_request == most
    assert plan.workspace_bytes >= plan.partial_offset + (most > 1) * len(items) * hq * 130 * 4


@pytest.mark.parametrize("pages,tail,hq,hkv", [
    ([1], [0], 32, 8), ([0], [0], 32, 8), ([3056], [16], 32, 8), ([0], [4000], 32, 8),
    ([0, 5, 0, 100000], [0, 0, 16, 16], 64, 4), ([256], [16], 32, 8), ([257], [0], 8, 8), ([512], [16], 32, 8)])
def test_plan_covers_every_page_once(pages, tail, hq, hkv):
    for cus in (1, 64, 256):
        _check_plan(pages, tail, hq, hkv, cus)


def test_plan_of_drawn_batches():
    rng = random.Random(11)
    for _ in range(200):
        n = rng.randint(1, 40)
        pages = [rng.choice([0, 1, rng.randint(0, 30), rng.randint(0, 6000)]) for _ in range(n)]
        tail = [rng.choice([0, 1, 16, rng.randint(0, 700)]) for _ in range(n)]
        hkv = rng.choice([1, 2, 5, 8, 16])
        _check_plan(pages, tail, hkv * rng.randint(1, 16), hkv, rng.choice([1, 100, 256, 304]))


@pytest.mark.parametrize("args,message", [
    (dict(indptr=[0, 4], num_qo_heads=30), "multiple of KV heads"),
    (dict(indptr=[0, 4], num_qo_heads=17, num_kv_heads=1), "at most 16 query heads"),
    (dict(indptr=[4, 0]), "non-decreasing"),
    (dict(indptr=[-1, 4]), "nonnegative"),
    (dict(indptr=[0, 4], tail_indptr=[0, -1]), "non-decreasing"),
    (dict(indptr=[0, 4], num_kv_heads=0), "positive multiple"),
    (dict(indptr=[0, 2 ** 31 - 1]), "too many pages"),
])
def test_plan_refuses(args, message):
    with pytest.raises(RuntimeError, match=message):
        int4.plan_work_items(**args)
    with pytest.raises(ValueError):
        int4.plan_work_items([0])
    with pytest.raises(ValueError):
        int4.plan_work_items([0, 4], [0, 4, 8])


def test_plan_struct_mirrors_the_header():
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "pagegauge_hip.h").read_text()
    body = re.search(r"typedef struct pg_int4_plan \{(.*?)\} pg_int4_plan_t;", text, re.S).group(1)
    fields = re.findall(r"(int32_t|int64_t)\s+([a-z_0-9]+);", body)
    assert [n for _, n in fields] == [n for n, _ in _capi.Int4Plan._fields_]
    sizes = {"int32_t": 4, "int64_t": 8}
    assert all(ctypes.sizeof(t) == sizes[c] for (c, _), (_, t) in zip(fields, _capi.Int4Plan._fields_))


def _half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


def _ids(n):
    return torch.zeros(n, dtype=torch.int32)


def _quantize(**over):
    codes, scales = int4.allocate_pages(2, 2, "cpu")
    a = dict(key=_half(20, 2, 128), value=_half(20, 2, 128), codes=codes, scales=scales)
    a.update(over)
    key, value, codes, scales = (a.pop(n) for n in ("key", "value", "codes", "scales"))
    int4.quantize_pages(key, value, codes, scales, **a)


@pytest.mark.parametrize("over,message", [
    (dict(value=_half(19, 2, 128)), "identical"),
    (dict(key=torch.zeros(20, 2, 128), value=torch.zeros(20, 2, 128)), "float16"),
    (dict(key=_half(20, 2, 64), value=_half(20, 2, 64)), "dense heads"),
    (dict(codes=torch.zeros(2, 2, 2, 1024)), "uint8"),
    (dict(scales=_half(2, 2, 32)), "4-bit scales"),
    (dict(key=_half(40, 2, 128), value=_half(40, 2, 128)), "do not fit"),
    (dict(page_ids=_ids(3)), "page_ids"),
    (dict(page_ids=torch.zeros(2, dtype=torch.int64)), "page_ids"),
    (dict(key_center=_half(2, 128)), "go together"),
    (dict(key_center=_half(2, 64), value_center=_half(2, 64)), "centers must be"),
    (dict(exact_page_ids=_ids(2)), "exact key/value pages"),
    (dict(exact_page_ids=_ids(2), exact_key=_half(1, 16, 2, 128), exact_value=_half(1, 8, 2, 128)),
     "exact_value"),
    (dict(), "current CUDA device"),
])
def test_quantize_refuses(over, message):
    with pytest.raises(ValueError, match=message):
        _quantize(**over)


@pytest.mark.parametrize("kwargs,message", [
    (dict(tokens=33), "at most 32 tokens"), (dict(tokens=-1), "at most"),
    (dict(page_ids=_ids(1), tokens=17), "at most 16"),
    (dict(key=_half(31, 2, 128)), "rows must be"),
    (dict(key=_half(1, 2, 128).expand(32, 2, 128)), "overlap"),
    (dict(value_center=_half(2, 128)), "go together"),
    (dict(), "current CUDA device"),
])
def test_dequantize_refuses(kwargs, message):
    codes, scales = int4.allocate_pages(2, 2, "cpu")
    with pytest.raises(ValueError, match=message):
        int4.dequantize_pages(codes, scales, **kwargs)


def _append(**over):
    codes, scales = int4.allocate_pages(2, 2, "cpu")
    a = dict(rotary=rotary.RotaryEmbedding(128, device="cpu"), query=_half(3, 8, 128),
             key=_half(3, 2, 128), value=_half(3, 2, 128), positions=_ids(3), exact_page_ids=_ids(3),
             code_page_ids=_ids(3), key_center=_half(3, 2, 128), value_center=_half(3, 2, 128),
             rotated_query=_half(3, 8, 128), exact_key=_half(4, 16, 2, 128),
             exact_value=_half(4, 16, 2, 128), codes=codes, scales=scales)
    a.update(over)
    int4.rope_append(**a)


@pytest.mark.parametrize("over,message", [
    (dict(rotary=rotary.RotaryEmbedding(64, device="cpu")), "128 dims"),
    (dict(query=_half(2, 8, 128)), "row per request"),
    (dict(value=_half(3, 1, 128)), "row per request"),
    (dict(positions=_ids(2)), "positions"),
    (dict(code_page_ids=_ids(6)[::2]), "code_page_ids"),
    (dict(key_center=None, value_center=None), "required"),
    (dict(key_center=_half(2, 128), value_center=_half(2, 128)), "centers must be"),
    (dict(rotated_query=_half(3, 8, 64)), "rotated_query"),
    (dict(exact_key=_half(4, 16, 1, 128)), "exact_key"),
    (dict(), "current CUDA device"),
])
def test_append_refuses(over, message):
    with pytest.raises(ValueError, match=message):
        _append(**over)


def test_decode_refuses_memory_of_the_host():
    with pytest.raises(ValueError, match="CUDA uint8"):
        int4.Int4PagedDecode(torch.zeros(1024, dtype=torch.uint8))


@pytest.mark.skipif(torch.cuda.is_available(), reason="host-only checks of the C entry points")
@pytest.mark.parametrize("name,args,code,message", [
    ("pg_int4_quantize_pages", (None, 1, 4096, 1, None, None, 4096, 4096, 1, None, None, None, None, 0,
                                16, 1, None), 1, "null tensor"),
    ("pg_int4_quantize_pages", (4096, 1, 4096, 1, None, None, 4097, 4096, 1, None, None, None, None, 0,
                                16, 1, None), 1, "16-byte aligned"),
    ("pg_int4_quantize_pages", (4096, 1, 4096, 1, 4096, None, 4096, 4096, 1, None, None, None, None, 0,
                                16, 1, None), 1, "go together"),
    ("pg_int4_quantize_pages", (4096, 1, 4096, 1, None, None, 4096, 4096, 1, None, 4096, None, None, 0,
                                16, 1, None), 1, "exact page ids"),
    ("pg_int4_quantize_pages", (4096, 1, 4096, 1, None, None, 4096, 4096, 1, None, None, None, None, 0,
                                1 << 50, 8, None), 3, "too many pages"),
    # fewer pages than a launch has workgroups, but not times two blocks of heads
    ("pg_int4_quantize_pages", (4096, 1, 4096, 1, None, None, 4096, 4096, 1, None, None, None, None, 0,
                                16 * 10 ** 7, 8, None), 3, "too many pages"),
    ("pg_int4_dequantize_pages", (4096, 4096, 1, None, None, None, 4096, 1, 4096, 1, 16 * 10 ** 7, 8, None),
     3, "too many pages"),
    ("pg_int4_dequantize_pages", (4096, 4096, 0, None, None, None, 4096, 1, 4096, 1, 16, 1, None), 1,
     "no pages"),
    ("pg_int4_dequantize_pages", (4096, 4096, 1, None, None, None, 4096, 1, 4096, 1, -1, 1, None), 1,
     "nonnegative"),
    ("pg_int4_rope_append", (4096, 4096, 4096, 1, 1, 1, 4096, 4096, ctypes.c_float(1.0), 130, 0, 4096,
                             4096, 4096, 4096, 4096, 4096, 4096, 1, 4096, 4096, 1, 1, 4, 1, None), 1,
     "even number"),
    ("pg_int4_rope_append", (4096, 4096, 4096, 1, 1, 1, 4096, 4096, ctypes.c_float(1.0), 128, 0, 4096,
                             4096, 4096, 4096, 4096, 4096, 4100, 1, 4096, 4096, 1, 1, 4, 1, None), 1,
     "16-byte aligned"),
    ("pg_int4_decode_run", (None, *([None] * 1), 0, *([None] * 9), 0, None, None, ctypes.c_float(0.1),
                            None, None), 1, "null run argument"),
])
def test_c_entry_points_refuse(name, args, code, message):
    rc = getattr(_capi.library(), name)(*args)
    assert rc == code and message in _capi.last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="host-only checks of the C entry points")
@pytest.mark.parametrize("over,message", [
    (dict(query=None), "null run argument"), (dict(codes=None), "history segment"),
    (dict(tail_k=None), "tail segment"), (dict(sm_scale=0.0), "sm_scale"),
    (dict(sm_scale=float("inf")), "sm_scale"), (dict(sm_scale=float("nan")), "sm_scale"),
    (dict(query=4104), "16-byte aligned"), (dict(scales=4100), "16-byte aligned"),
    (dict(stride=4), "16-byte aligned"), (dict(center=4098), "4-byte aligned"),
    (dict(heads=0), "not one of")])
def test_decode_run_refuses(over, message):
    plan, _, _ = int4.plan_work_items([0, 40], [0, 16])
    a = dict(query=4096, stride=4096, codes=4096, scales=4096, indices=4096, last=4096, tail_k=4096,
             tail_v=4096, tail_indices=4096, tail_last=4096, center=None, center_stride=0, out=4096,
             lse=None, sm_scale=0.1, workspace=4096, stream=None)
    a.update(over)
    if "heads" in a:
        plan.num_kv_heads = a.pop("heads")
    a["sm_scale"] = ctypes.c_float(a["sm_scale"])
    rc = _capi.library().pg_int4_decode_run(ctypes.byref(plan), *a.values())
    assert rc == 1 and message in _capi.last_error()


def test_last_lengths_are_checked_where_there_are_pages():
    indptr = torch.tensor([0, 2, 2, 3])
    int4._check_last(indptr, torch.tensor([16, 99, 1]), "last")
    for bad in ([0, 1, 1], [17, 1, 1], [1, 1, -1]):
        with pytest.raises(ValueError, match="last must lie"):
            int4._check_last(indptr, torch.tensor(bad), "last")


def _weights(pages, tail, hq, hkv, cus):
    tables = [np.concatenate(([0], np.cumsum(n))).tolist() for n in (pages, tail)]
    _, items, _ = int4.plan_work_items(*tables, hq, hkv, cus)
    return [(i[2] - i[1]) + 4 * (i[5] - i[4]) for i in items.tolist()]


def _check_shares(pages, tail, hkv, cus):
    """No item outweighs both two full ones and twice an even share (and the tail page
    that a cut falls into)."""
    share = -(-(sum(pages) + 4 * sum(tail)) // max(len(pages), cus // hkv, 1))
    assert max(_weights(pages, tail, 4 * hkv, hkv, cus)) <= max(2 * 256, 2 * share) + 4


@pytest.mark.parametrize("pages,tail", [
    # a long exact tail beside a history that needs more items than there are CUs
    ([100000, 0], [0, 4000]), ([100000, 200], [16, 4000]),
    # and beside so many requests that each would be one item
    ([40] * 299 + [0], [0] * 299 + [3000]), ([240] * 256 + [16], [16] * 256 + [1000])])
def test_long_tails_are_shared_out(pages, tail):
    _check_shares(pages, tail, 8, 256)


def test_shares_of_drawn_batches():
    rng = random.Random(12)
    for _ in range(200):
        n = rng.choice([1, 2, 7, rng.randint(1, 400)])
        pages = [rng.choice([0, rng.randint(0, 256), rng.randint(0, 20000)]) for _ in range(n)]
        tail = [rng.choice([0, 16, rng.randint(0, 200), rng.randint(0, 5000)]) for _ in range(n)]
        _check_shares(pages, tail, rng.choice([1, 2, 8, 16]), rng.choice([64, 256, 304]))


@pytest.mark.parametrize("pages,tail,items", [
    # one item per CU: 49K and 64K tokens; two where its waves cannot hold its pages
    # (128K tokens and a ring) or requests do not divide over so few (17 of 3.3K)
    ([3056], [16], 32), ([4080], [16], 32), ([8192], [16], 64), ([192] * 17, [16] * 17, 51),
    ([512] * 16, [0] * 16, 32),
    # whole requests, one item each
    ([144] * 256, [16] * 256, 256)])
def test_plans_take_the_items_that_the_rules_say(pages, tail, items):
    assert len(_weights(pages, tail, 32, 8, 256)) == items


@pytest.mark.parametrize("pages,tail", [([100000, 0], [0, 600000]), ([0] * 10000, [3000000] + [0] * 9999)])
def test_long_tails_keep_to_the_items_of_a_request(pages, tail):
    """Tails of millions of tokens are shared out among as many items as a request may have."""
    tables = [np.concatenate(([0], np.cumsum(n))).tolist() for n in (pages, tail)]
    plan, items, _ = int4.plan_work_items(*tables)
    assert 2048 < plan.max_items_per_request <= 4096
    assert int(items[:, 5].max()) == sum(tail)


@pytest.mark.parametrize("name", ["scales", "key_center", "value_center"])
def test_dequantize_refuses_gradients(name):
    """The result would have no history: it is not computed, but for no_grad()."""
    codes, scales = int4.allocate_pages(2, 2, "cpu")
    a = dict(scales=scales, key_center=_half(2, 128), value_center=_half(2, 128))
    a[name].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        int4.dequantize_pages(codes, **a)
    with torch.no_grad(), pytest.raises(ValueError, match="current CUDA device"):
        int4.dequantize_pages(codes, **a)
