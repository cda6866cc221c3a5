"""Attention over the cache held in 4 bits, where a wave takes many groups of pages, a
workgroup many exact pages and a join many items: plans for few CUs and for long
requests, whose items are asserted before the results (bounds: test_gpu_int4_decode)."""

from __future__ import annotations

import pytest
import torch

from test_gpu_int4_decode import Case, both_forms

pytestmark = pytest.mark.gpu


def _planned(cuda, history, tail, kv_heads, group, num_cus):
    """(the case, its items [n, 8]), planned for so many CUs."""
    from pagegauge_amd import int4

    c = Case(cuda, history, tail, kv_heads, group)
    (indptr, _, _), (tail_indptr, _, _) = c.tables
    heads = dict(num_qo_heads=kv_heads * group, num_kv_heads=kv_heads, num_cus=num_cus)
    c.decode.plan(*c.tables[0], *c.tables[1], **heads)
    _, items, _ = int4.plan_work_items(indptr, tail_indptr, **heads)
    assert c.decode.num_work_items == len(items)
    return c, items


# 9 to 64 groups of 4 pages for 4 waves, odd and even numbers of them per wave, the last
# one short of pages, the last page short of tokens
@pytest.mark.parametrize("pages", [33, 47, 48, 49, 65, 100, 129, 255, 256])
@pytest.mark.parametrize("missing", [0, 5])
@both_forms
def test_items_of_many_groups(cuda, pages, missing, kv_heads, group):
    print(f"attention item of {pages} pages less {missing} tokens heads={kv_heads}x{group}", flush=True)
    c, items = _planned(cuda, [16 * pages - missing], [0], kv_heads, group, 1)
    assert len(items) == 1 and int(items[0, 2] - items[0, 1]) == pages
    c.check(*c.run())


@both_forms
def test_past_the_pages_of_an_item(cuda, kv_heads, group):
    """257 pages, two items; beside requests of one item that are short, empty and full."""
    c, items = _planned(cuda, [4110, 9, 0, 4096], [0, 0, 20, 0], kv_heads, group, 1)
    assert [int(n) for n in items[:, 7]] == [2, 2, 1, 1, 1]
    assert int((items[:, 2] - items[:, 1]).max()) == 256
    c.check(*c.run())


# 9 to 40 exact pages for 4 waves of 2 at a time, alone and behind a history of 1 and of
# several groups per wave
@pytest.mark.parametrize("tail", [9 * 16, 10 * 16 - 7, 16 * 16, 17 * 16 - 1, 31 * 16, 40 * 16 - 15])
@pytest.mark.parametrize("history", [0, 16, 30 * 16 - 3, 100 * 16])
@both_forms
def test_items_of_many_exact_pages(cuda, history, tail, kv_heads, group):
    print(f"attention item of {history} + {tail} tokens heads={kv_heads}x{group}", flush=True)
    c, items = _planned(cuda, [history], [tail], kv_heads, group, 1)
    assert len(items) == 1 and int(items[0, 5] - items[0, 4]) == -(-tail // 16)
    c.check(*c.run())


# more than the 64 items that a join requests together, and more than twice as many
@pytest.mark.parametrize("pages,tail", [(1070, 0), (1100, 250), (2150, 16)])
@pytest.mark.parametrize("group", [4, 16])
def test_joins_of_many_items(cuda, pages, tail, group):
    print(f"attention of {pages} pages + {tail} tokens, 1 x {group} heads", flush=True)
    c, items = _planned(cuda, [16 * pages - 9], [tail], 1, group, 256)
    assert len(items) > (128 if pages > 2048 else 64)
    c.check(*c.run())
    # and joined beside a request of one item
    c, items = _planned(cuda, [30, 16 * pages], [0, tail], 1, group, 256)
    assert int(items[0, 7]) == 1 and len(items) > 65
    c.check(*c.run())


def test_scores_that_rise_along_an_item(cuda):
    """The softmax's base moves in every group of a wave, and a join's from item to item."""
    for num_cus in (1, 256):
        c, items = _planned(cuda, [4096], [100], 2, 4, num_cus)
        assert (len(items) == 1) == (num_cus == 1)
        ids = c.tables[0][1].long()
        # keys' scales grow with the page, and one code's sign goes with the query's
        c.codes[:, :, 0] = 0x99                      # every key code 1
        c.q.abs_()
        c.scales[ids, :, :, 0] = (torch.arange(1, 257, device=cuda) / 64.0).half()[:, None, None, None]
        c.check(*c.run())
