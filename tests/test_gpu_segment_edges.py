"""Attention over shared prefixes and selected pages where a call is allowed and rare:
pages without a token left, tables that lose pages after the plan, scores of any size
(tolerances: segment_helpers).

A prefix of up to 32 query rows per KV head takes the form without tiles, of up to 64 the
one with tiles of two waves' rows, of more the one of four."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import test_gpu_sparse as selecting
from segment_helpers import LOG2E, Batch, check_head, values
from test_gpu_prefix import both_kinds, planned, run, spread

pytestmark = pytest.mark.gpu

# of 4 heads per KV head: 8 and 24 rows, 36, 80 and 160
FORMS = [2, 6, 9, 20, 40]


@pytest.mark.parametrize("requests", FORMS)
@pytest.mark.parametrize("left", [float("nan"), float("inf"), 65504.0])
def test_a_page_without_tokens_weighs_nothing(cuda, requests, left):
    """Whatever its scales are: lengths may move to 0, and such a page was never written."""
    print(f"no tokens {requests} {left}", flush=True)
    b = Batch(cuda, [(0, requests, 1000)], spread(requests, 17, 70), [0] * requests, 1, 4, scale=2.0 ** -13)
    decode = planned(b, cuda)
    b.prefix_last.zero_()
    b.last.zero_()
    out, lse = run(decode, b)
    b.check(out, lse)
    pages = torch.cat((b.prefix_ids[-1:], b.ids[(b.own_ptr[1:] - 1).long().to(cuda)])).long()
    for scale in b.scales:
        scale[pages] = left
    got, got_lse = run(decode, b)
    assert torch.equal(got, out) and torch.equal(got_lse, lse)


def cleared(ids, every, first):
    """Ids with some entries below 0."""
    ids = ids.clone()
    ids[first::every] = -1
    ids[first + every::3 * every] = -2 ** 31
    return ids


def with_a_spoiled_first_page(b):
    """The pools with a page in front that no table names, and holds what must not count."""
    for pools in (b.cache, b.exact):
        for i in range(2):
            bad = torch.full_like(pools[i][:1], 77 if pools[i].dtype is torch.int8 else float("nan"))
            pools[i] = torch.cat((bad, pools[i]))
    if b.kind is torch.int8:
        b.scales = [torch.cat((torch.full_like(s[:1], float("nan")), s)) for s in b.scales]
    for ids in (b.prefix_ids, b.ids, b.tail_ids):
        ids += 1


def seen_of(b, selected=None):
    """``f(b, h)``: float64 K and V [T, 128] that KV head h of request b sees, without the
    entries below 0."""
    pools = [values(c, s) for c, s in zip(b.cache, b.scales)]
    exact = [values(c, None) for c in b.exact]

    def rows(pools, ptr, ids, last, i, h, positions=None):
        table, n = ids[int(ptr[i]):int(ptr[i + 1])].tolist(), int(last[i])
        return [[p[page, :n if at == len(table) - 1 else 16, h] for p in pools] for at, page in enumerate(table)
                if page >= 0 and (positions is None or at in positions)]

    def seen(r, h):
        found = []
        for i, (first, end, _) in enumerate(b.segments):
            if first <= r < end:
                found += rows(pools, b.prefix_ptr, b.prefix_ids, b.prefix_last, i, h)
        found += rows(pools, b.own_ptr, b.ids, b.last, r, h, None if selected is None else selected[r, h].tolist())
        found += rows(exact, b.tail_ptr, b.tail_ids, b.tail_last, r, h)
        return [np.concatenate([x[i] for x in found] + [np.zeros((0, 128))]) for i in range(2)]

    return seen


def check(b, out, lse, seen, single_part=True):
    for r in range(b.batch):
        for h in range(b.hkv):
            rows = slice(h * b.group, (h + 1) * b.group)
            check_head(out[r, rows].double().cpu().numpy(), lse[r, rows].double().cpu().numpy(),
                       b.q[r, rows].cpu().numpy(), *seen(r, h), b.center[r, h].cpu().numpy(), 128 ** -0.5, single_part)


@both_kinds
@pytest.mark.parametrize("requests", FORMS)
def test_entries_below_0_are_no_pages(cuda, requests, kind):
    """Rewritten in place after the plan: some, all of a tile, the last ones, all."""
    print(f"no pages {requests} {kind}", flush=True)
    b = Batch(cuda, [(0, requests, 3005), (1, requests, 90)], spread(requests, 1, 300), spread(requests, 0, 60), 2, 4,
              kind)
    with_a_spoiled_first_page(b)
    decode = planned(b, cuda)
    whole = [t.clone() for t in (b.prefix_ids, b.ids, b.tail_ids)]
    last = b.prefix_ids.clone()
    last[int(b.prefix_ptr[1]) - 1] = last[-1] = -1
    tile = b.prefix_ids.clone()
    tile[16:25] = -1
    for prefix_ids, ids, tail_ids in ((cleared(whole[0], 7, 2), cleared(whole[1], 3, 1), cleared(whole[2], 2, 0)),
                                      (tile, whole[1], whole[2]), (last, cleared(whole[1], 1, 0), whole[2]),
                                      [torch.full_like(t, -1) for t in whole]):
        for at, new in zip((b.prefix_ids, b.ids, b.tail_ids), (prefix_ids, ids, tail_ids)):
            at.copy_(new)
        out, lse = run(decode, b)
        check(b, out, lse, seen_of(b))
    assert bool((lse == -torch.inf).all())
    again = planned(b, cuda)                                 # and planned with such entries
    assert torch.equal(run(again, b)[0], out)


@pytest.mark.parametrize("group", [4, 16])
@pytest.mark.parametrize("pages", [9, 200])
def test_selections_leave_out_entries_below_0(cuda, pages, group):
    print(f"selected no pages {pages} {group}", flush=True)
    b = Batch(cuda, [], [3000, 100, 1, 1601], [40, 0, 16, 3], 2, group)
    with_a_spoiled_first_page(b)
    bounds = selecting.bounds_of(b, cuda)
    bounds[0, :, 0], bounds[0, :, 1] = -128, 127
    decode = selecting.planned(b, cuda, pages, 1, 1)
    for every, first in ((5, 3), (1, 0)):
        b.ids.copy_(cleared(b.ids, every, first))
        b.ids[int(b.own_ptr[1]) - 1] = -1                    # a forced one among them
        selected = decode.select(b.q, bounds, b.scales[0])
        want = np.full((4, 2, pages), -1)
        for r in range(4):
            at = b.ids[int(b.own_ptr[r]):int(b.own_ptr[r + 1])]
            s = selecting.expected_scores(b.q[r], bounds[at.clamp(min=0).long()], b.scales[0][at.clamp(min=0).long()],
                                          group)
            s[:, at.cpu().numpy() < 0] = -np.inf
            s[:, 0] = s[:, -1] = np.inf
            for h in range(2):
                best = sorted(np.argsort(-s[h], kind="stable")[:pages])
                want[r, h, :len(best)] = best
        assert np.array_equal(selected.cpu().numpy(), want)
        out, lse = selecting.run(decode, b, selected)
        check(b, out, lse, seen_of(b, selected.cpu().numpy()), single_part=False)


def test_ended_requests_and_a_pool_cut_to_its_pages(cuda, monkeypatch):
    """Requests end, the pool is compacted, tables are rewritten in place and the planes cut to
    what is in use: the others' attention keeps its bits, and with ids checked, those past a
    cut are refused."""
    from pagegauge_amd import decode as checks
    from pagegauge_amd import pages

    monkeypatch.setattr(checks, "CHECK_PAGE_IDS", True)
    b = Batch(cuda, [(0, 12, 700)], spread(12, 20, 200), [0] * 12, 2, 4)
    count = len(b.cache[0])
    pool = pages.PagePool(count, device=cuda)
    pool.share(b.prefix_ids)
    pool.share(b.ids)
    bounds = selecting.bounds_of(b, cuda)
    decode, part = planned(b, cuda, with_tail=False), selecting.planned(b, cuda, 5, with_tail=False)
    out, lse = run(decode, b, exact_cache=None)
    selected = part.select(b.q, bounds, b.scales[0])
    part_out = selecting.run(part, b, selected, exact_cache=None)
    for r in (0, 5):
        pool.release(b.ids[int(b.own_ptr[r]):int(b.own_ptr[r + 1])].contiguous())
    moves = pool.stage_compaction()
    planes = (*b.cache, *b.scales, bounds)
    pages.copy_pages(planes, moves.source, moves.target)
    for ids in (b.prefix_ids, b.ids):
        pages.rewrite_ids(ids, moves.remap, out=ids)
    pool.commit_compaction(moves)
    live = int(moves.live)
    assert live < count and bool((b.ids < 0).any())
    b.cache, b.scales, bounds = [c[:live].clone() for c in b.cache], [s[:live].clone() for s in b.scales], bounds[:live]
    got, got_lse = run(decode, b, exact_cache=None)
    got_selected = part.select(b.q, bounds, b.scales[0])
    got_part = selecting.run(part, b, got_selected, exact_cache=None)
    stay = [r for r in range(12) if r not in (0, 5)]
    for x, y in ((got, out), (got_lse, lse), (got_selected, selected), *zip(got_part, part_out)):
        assert torch.equal(x[stay], y[stay])
    check(b, got, got_lse, seen_of(b))
    for cut, message in ((int(b.ids.max()), "page ids span"), (0, "no pages")):
        less = dict(kv_cache=[c[:cut] for c in b.cache], k_page_scale=b.scales[0][:cut], v_page_scale=b.scales[1][:cut])
        with pytest.raises(ValueError, match=message):
            run(decode, b, exact_cache=None, **less)
        with pytest.raises(ValueError, match=message):
            part.select(b.q, bounds[:cut], b.scales[0][:cut])


@both_kinds
@pytest.mark.parametrize("requests", FORMS)
@pytest.mark.parametrize("sm_scale", [2.0 ** -60, 128 ** -0.5, 2.0 ** 30, float(np.nextafter(np.float32(2.0 ** 80), 0.0))])
def test_scores_of_any_size(cuda, requests, kind, sm_scale):
    """Queries of +-2^15 meet keys that are the same in all dims: every score is exact and they
    are equal or at least 2^6 apart in base 2, or with the smallest softmax scale within 2^-16
    of each other.  A row sees the mean of the values at its largest score, or of all."""
    print(f"scores {requests} {kind} {sm_scale}", flush=True)
    b = Batch(cuda, [(0, requests, 1000)], spread(requests, 17, 70), spread(requests, 0, 40), 1, 4, kind)
    gen = torch.Generator().manual_seed(3)
    b.q = (torch.randint(0, 2, (requests, 4, 1), generator=gen) * 2 - 1).expand(requests, 4, 128).half() * 2.0 ** 15
    b.q = b.q.contiguous().to(cuda)
    pool = len(b.cache[0])
    sign = (torch.randint(0, 5, (pool, 16, 1, 1), generator=gen) == 0).expand(pool, 16, 1, 128).to(cuda)
    if kind is torch.int8:
        b.cache[0] = torch.where(sign, 127, -128).to(torch.int8)
        b.scales[0].fill_(2.0 ** 15)
    else:
        b.cache[0] = torch.where(sign, 2.0 ** 15, -2.0 ** 14).half()
    pages = len(b.exact[0])
    b.exact[0] = torch.where(sign.repeat(2, 1, 1, 1)[:pages] if pages > pool else sign[:pages], 2.0 ** 15, 2.0 ** 9).half()
    out, lse = run(planned(b, cuda), b, sm_scale=sm_scale)
    seen = b.keys_and_values()
    for r in range(requests):
        k, v = seen(r, 0)
        for row in range(4):
            s = b.q[r, row].double().cpu().numpy() @ k.T * (np.float64(np.float32(sm_scale)) * LOG2E)
            weight = np.exp2(s - s.max())
            want = weight @ v / weight.sum() + b.center[r, 0].double().cpu().numpy()
            # a weight is 1, 0 or off by 2^-14 of itself; two-part probabilities are off by 2^-20,
            # one-part ones by 2^-11, sums by T / 16 + 64 float32 roundings
            bound = (2.0 ** -13 + 2.0 ** -11 + len(k) * 2.0 ** -28) * np.abs(v).max()
            got = out[r, row].double().cpu().numpy()
            assert (np.abs(got - want) <= bound + np.abs(want) * 2.0 ** -11 + 2.0 ** -24).all(), (r, row)
            want_lse = s.max() + np.log2(weight.sum())
            assert abs(float(lse[r, row]) - want_lse) <= 2.0 ** -21 * abs(want_lse) + 2.0 ** -12, (r, row)


def test_softmax_scales_past_float32_are_refused(cuda):
    """Scores of INT8 pages reach 2^46, times 2^80 and log2(e) still float32."""
    b = Batch(cuda, [(0, 2, 40)], [20, 3], [5, 5], 2, 4)
    decode = planned(b, cuda)
    for sm_scale in (2.0 ** 80, 2.0 ** 99):
        with pytest.raises(RuntimeError, match="sm_scale"):
            run(decode, b, sm_scale=sm_scale)


def test_selected_pages_with_scores_of_any_size(cuda):
    """Codes, scales and queries at their largest: the exact tail's scores are far below."""
    b = Batch(cuda, [], [1000, 90], [40, 0], 1, 4)
    b.q = torch.full_like(b.q, 2.0 ** 15)
    b.cache[0].fill_(-128)
    b.cache[0][b.ids[::2].long()] = 127
    b.scales[0].fill_(2.0 ** 15)
    decode = selecting.planned(b, cuda, 8)
    selected = decode.select(b.q, selecting.bounds_of(b, cuda), b.scales[0])
    for sm_scale in (128 ** -0.5, 2.0 ** 79):
        out, lse = selecting.run(decode, b, selected, sm_scale=sm_scale)
        seen = b.keys_and_values(selected.cpu().numpy())
        for r in range(2):
            k, v = seen(r, 0)
            top = k[:, 0] == k[:, 0].max()
            want = v[top].mean(0) + b.center[r, 0].double().cpu().numpy()
            got = out[r].double().cpu().numpy()
            assert (np.abs(got - want) <= 2.0 ** -10 * np.abs(v).max() + np.abs(want) * 2.0 ** -11).all()
            s = 128 * 2.0 ** 15 * k[:, 0].max() * np.float64(np.float32(sm_scale)) * LOG2E
            assert np.allclose(lse[r].cpu().numpy(), s + np.log2(top.sum()), rtol=2.0 ** -21, atol=0)
