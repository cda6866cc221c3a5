"""Bounds, scores and choice of pages to the bit, and attention over selected pages
against float64 (tolerances: segment_helpers)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from segment_helpers import Batch

pytestmark = pytest.mark.gpu


def planned(b, cuda, pages, first=1, last=1, with_tail=True, workspace_bytes=64 << 20):
    from pagegauge_amd import sparse

    decode = sparse.SelectedPagesDecode(torch.empty(workspace_bytes, device=cuda, dtype=torch.uint8))
    decode.plan(*b.own_table(), *(b.tail_table() if with_tail else ()), pages=pages, first_pages=first,
                last_pages=last, num_qo_heads=b.hkv * b.group, num_kv_heads=b.hkv)
    return decode


def run(decode, b, selected, **over):
    a = dict(q=b.q, kv_cache=b.cache, k_page_scale=b.scales[0], v_page_scale=b.scales[1], selected=selected,
             exact_cache=b.exact, value_center=b.center, return_lse=True)
    a.update(over)
    return decode.run(**a)


def bounds_of(b, cuda):
    from pagegauge_amd import sparse

    bounds = sparse.allocate_bounds(len(b.cache[0]), b.hkv, cuda)
    sparse.key_bounds(b.cache[0], bounds)
    return bounds


def expected_scores(q, bounds, scale, group):
    """float32 [Hkv, pages] as the C header states them."""
    q, bounds = q.cpu().numpy().astype(np.float64), bounds.cpu().numpy().astype(np.int64)
    scale = scale.cpu().numpy().astype(np.float32)
    scores = np.full((bounds.shape[1], len(bounds)), -np.inf, np.float32)
    for row, values in enumerate(q):
        h = row // group
        if not np.isfinite(values).all():
            continue
        largest = np.abs(values).max()
        x = int(np.frexp(largest)[1]) if largest else 0
        steps = np.clip(np.rint(np.ldexp(values, 7 - x)), -127, 127).astype(np.int64)
        low, high = bounds[:, h, 0], bounds[:, h, 1]
        total = np.maximum(steps * low, steps * high).sum(1)
        # where a page without tokens has low > high, the least is on the other side
        total = np.where((low > high).any(1), (np.maximum(steps, 0) * high + np.minimum(steps, 0) * low).sum(1), total)
        with np.errstate(all="ignore"):
            s = np.float32(total) * scale[:, h] * np.float32(2.0 ** (x - 7))
        scores[h] = np.maximum(scores[h], np.where(np.isnan(s), np.float32(-np.inf), s))
    return scores


def expected_selection(b, bounds, pages, first, last):
    ids, found = b.ids.cpu(), np.full((b.batch, b.hkv, pages), -1)
    for i in range(b.batch):
        at = ids[b.own_ptr[i]:b.own_ptr[i + 1]].long().to(bounds.device)
        s = expected_scores(b.q[i], bounds[at], b.scales[0][at], b.group)
        s[:, :first] = np.inf
        s[:, max(0, len(at) - last):] = np.inf
        for h in range(b.hkv):
            best = sorted(np.argsort(-s[h], kind="stable")[:pages])
            found[i, h, :len(best)] = best
    return found


@pytest.mark.parametrize("kv_heads", [1, 3, 8])
def test_bounds(cuda, kv_heads):
    from pagegauge_amd import sparse

    gen = torch.Generator().manual_seed(1)
    codes = torch.randint(-128, 128, (77, 16, kv_heads, 128), generator=gen).to(torch.int8).to(cuda)
    codes[5] = -128
    codes[6] = 127
    bounds = sparse.allocate_bounds(77, kv_heads, cuda)
    sparse.key_bounds(codes, bounds)
    assert torch.equal(bounds[:, :, 0], codes.amin(1)) and torch.equal(bounds[:, :, 1], codes.amax(1))
    ids = torch.tensor([3, -1, 70, 77, 5, 0, 2 ** 31 - 1, 9], dtype=torch.int32, device=cuda)
    lengths = torch.tensor([1, 16, 7, 4, 0, 16, 2, 99], dtype=torch.int32, device=cuda)
    got = torch.full_like(bounds, 11)
    sparse.key_bounds(codes, got, page_ids=ids, lengths=lengths)
    want = torch.full_like(bounds, 11)
    for page, n in ((3, 1), (70, 7), (0, 16), (9, 16)):
        want[page, :, 0], want[page, :, 1] = codes[page, :n].amin(0), codes[page, :n].amax(0)
    want[5, :, 0], want[5, :, 1] = 127, -128
    assert torch.equal(got, want)
    sparse.key_bounds(codes, got, page_ids=ids[:0])
    assert torch.equal(got, want)


# fewer pages than are taken, as many, one more, several stretches of the choice
@pytest.mark.parametrize("own", [[1], [16 * 8], [16 * 9], [16 * 9 + 5], [300, 0, 5000, 129, 17], [16 * 2500 + 1]])
@pytest.mark.parametrize("first,last", [(0, 0), (1, 1), (3, 5)])
@pytest.mark.parametrize("kv_heads,group", [(2, 4), (3, 1), (1, 16), (2, 7)])
def test_choice(cuda, own, first, last, kv_heads, group):
    print(f"choice {own} {first} {last} {kv_heads}x{group}", flush=True)
    b = Batch(cuda, [], own, [0] * len(own), kv_heads, group)
    bounds = bounds_of(b, cuda)
    got = planned(b, cuda, 8, first, last, with_tail=False).select(b.q, bounds, b.scales[0])
    assert np.array_equal(got.cpu().numpy(), expected_selection(b, bounds, 8, first, last))


@pytest.mark.parametrize("pages", [1, 64, 500, 1999])
def test_choice_of_many(cuda, pages):
    b = Batch(cuda, [], [32000, 9000], [0, 0], 2, 4)
    bounds = bounds_of(b, cuda)
    first = min(1, pages - 1)
    got = planned(b, cuda, pages, first, 1, with_tail=False).select(b.q, bounds, b.scales[0])
    assert np.array_equal(got.cpu().numpy(), expected_selection(b, bounds, pages, first, 1))


@pytest.mark.parametrize("pages", [2047, 5003, 20_011, 100_003])
@pytest.mark.parametrize("alike", [True, False])
def test_choice_among_many_pages(cuda, pages, alike):
    """Bounds alone, of long contexts, with equal scores throughout or hardly any."""
    from pagegauge_amd import sparse

    print(f"choice among {pages} {alike}", flush=True)
    gen = torch.Generator().manual_seed(9)
    bounds = torch.randint(-2, 3, (pages, 1, 2, 128), generator=gen).to(torch.int8).to(cuda)
    bounds[:, :, 1] += 4
    if alike:
        bounds[:, :, :, 4:] = 0
    scale = torch.ones(pages, 1, dtype=torch.float16, device=cuda)
    if not alike:
        scale = (torch.rand(pages, 1, generator=gen) + 0.5).half().to(cuda)
    q = torch.zeros(1, 2, 128, dtype=torch.float16, device=cuda)
    q[0, 0, :4], q[0, 1, 1:3] = 1.0, -0.5
    ids = torch.randperm(pages, generator=gen).int().to(cuda)
    decode = sparse.SelectedPagesDecode(torch.empty(64 << 20, device=cuda, dtype=torch.uint8))
    decode.plan([0, pages], ids, torch.tensor([16], dtype=torch.int32, device=cuda), pages=777, num_qo_heads=2,
                num_kv_heads=1)
    got = decode.select(q, bounds, scale).cpu().numpy()
    s = expected_scores(q[0], bounds[ids.long()], scale[ids.long()], 2)
    s[0, 0] = s[0, -1] = np.inf
    assert (len(np.unique(s)) < 60) == alike
    assert np.array_equal(got[0, 0], sorted(np.argsort(-s[0], kind="stable")[:777]))


def test_choice_without_a_say(cuda):
    """Zero queries, spoiled ones, equal bounds, pages without tokens, spoiled scales."""
    b = Batch(cuda, [], [2000, 3000, 1500, 1600], [0] * 4, 2, 4)
    b.q[0, :4] = 0                                        # ties: the lowest positions
    b.q[1, 0, 3], b.q[1, 2, 5] = float("nan"), float("inf")
    b.q[2, 4:] = float("nan")                             # no row has a say
    b.q[3] *= 2.0 ** -14                                  # subnormal values
    bounds = bounds_of(b, cuda)
    bounds[b.ids[int(b.own_ptr[3]) + 20].long(), :, 0], bounds[b.ids[int(b.own_ptr[3]) + 20].long(), :, 1] = 127, -128
    at = b.ids[int(b.own_ptr[1]):].long()
    b.scales[0][at[7]], b.scales[0][at[9]] = float("nan"), float("inf")
    b.scales[0][at[11]] = 0
    got = planned(b, cuda, 30, 0, 2, with_tail=False).select(b.q, bounds, b.scales[0]).cpu().numpy()
    want = expected_selection(b, bounds, 30, 0, 2)
    assert np.array_equal(got, want)
    assert got[0, 0].tolist() == list(range(28)) + [123, 124]
    assert got[2, 1].tolist() == list(range(28)) + [92, 93]


@pytest.mark.parametrize("kv_heads,group", [(8, 4), (2, 16), (1, 1), (3, 7)])
@pytest.mark.parametrize("pages", [1, 6, 100, 700])
def test_attention_over_the_choice(cuda, kv_heads, group, pages):
    print(f"sparse {kv_heads}x{group} {pages}", flush=True)
    own, tail = [3000, 0, 90, 17, 1601, 1], [100, 16, 0, 1, 40, 0]
    b = Batch(cuda, [], own, tail, kv_heads, group)
    first = min(1, pages - 1)
    decode = planned(b, cuda, pages, first, 1)
    selected = decode.select(b.q, bounds_of(b, cuda), b.scales[0])
    b.check(*run(decode, b, selected), selected=selected.cpu().numpy(), single_part=False)
    without = planned(b, cuda, pages, first, 1, with_tail=False)
    out, lse = run(without, b, selected, exact_cache=None, value_center=None)
    b.tail_ptr.zero_()
    b.check(out, lse, selected=selected.cpu().numpy(), center=False, single_part=False)


def test_many_requests(cuda):
    """More than 1024 (request, head) pairs, ragged, some without a page."""
    gen = torch.Generator().manual_seed(4)
    own = torch.randint(0, 900, (150,), generator=gen).tolist()
    own[3] = own[149] = 0
    b = Batch(cuda, [], own, torch.randint(0, 40, (150,), generator=gen).tolist(), 2, 4)
    bounds = bounds_of(b, cuda)
    decode = planned(b, cuda, 20, 2, 1)
    selected = decode.select(b.q, bounds, b.scales[0])
    assert np.array_equal(selected.cpu().numpy(), expected_selection(b, bounds, 20, 2, 1))
    b.check(*run(decode, b, selected), selected=selected.cpu().numpy(), single_part=False)


def test_attention_over_a_callers_choice(cuda):
    """Any order; positions outside a table are not read; lengths move."""
    b = Batch(cuda, [], [1000, 40, 0, 333], [10, 0, 0, 0], 2, 4)
    gen = torch.Generator().manual_seed(8)
    selected = torch.full((4, 2, 9), -1, dtype=torch.int32)
    for i, pages in ((0, 63), (3, 21)):
        for h in range(2):
            selected[i, h] = torch.randperm(pages, generator=gen)[:9].int()
    selected[0, 0, 3], selected[0, 1, 0], selected[3, 0, 8] = 63, -5, 2 ** 31 - 1
    selected[0, 0, 5] = 62                                # the partial last page, inside the list
    selected[1, :, :3] = torch.tensor([2, 0, 1])
    decode = planned(b, cuda, 9, 0, 0)
    got = selected.to(cuda)
    b.check(*run(decode, b, got), selected=selected.numpy(), single_part=False)
    b.last.copy_(torch.tensor([1, 16, 0, 0]))
    b.check(*run(decode, b, got), selected=selected.numpy(), single_part=False)
    nothing = torch.full_like(got, -1)
    out, lse = run(decode, b, nothing)
    b.check(out, lse, selected=nothing.cpu().numpy(), single_part=False)
    assert bool((lse[1] == -torch.inf).all())


def test_captured_steps_follow_their_inputs(cuda):
    b = Batch(cuda, [], [5000, 600, 17], [40, 3, 16], 2, 4)
    bounds = bounds_of(b, cuda)
    decode = planned(b, cuda, 24)
    selected = decode.select(b.q, bounds, b.scales[0])
    out, lse = run(decode, b, selected)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode.select(b.q, bounds, b.scales[0], out=selected)
        run(decode, b, selected, out=out, lse=lse)
    gen = torch.Generator().manual_seed(5)
    for _ in range(4):
        b.q.copy_(torch.randn(b.q.shape, generator=gen))
        b.last.clamp_(max=int(torch.randint(1, 17, (1,), generator=gen)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(selected.cpu().numpy(), expected_selection(b, bounds, 24, 1, 1))
        want, want_lse = run(decode, b, selected.clone())
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_calls_on_another_stream(cuda):
    b = Batch(cuda, [], [4000, 90], [5, 5], 2, 4)
    bounds = bounds_of(b, cuda)
    decode = planned(b, cuda, 10)
    want = run(decode, b, decode.select(b.q, bounds, b.scales[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(decode, b, decode.select(b.q, bounds, b.scales[0]))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refuses(cuda):
    from pagegauge_amd import sparse

    b = Batch(cuda, [], [400, 90], [5, 5], 2, 4)
    bounds = bounds_of(b, cuda)
    for over, message in ((dict(pages=0, first=0, last=0), "at least one"), (dict(pages=3, first=2, last=2), "do not fit"),
                          (dict(pages=3, first=-1), "do not fit")):
        with pytest.raises(ValueError, match=message):
            planned(b, cuda, **over)
    decode = planned(b, cuda, 4)
    selected = decode.select(b.q, bounds, b.scales[0])
    for q, x, s, message in ((b.q.float(), bounds, b.scales[0], "float16"), (b.q, bounds[:, :1], b.scales[0], "bounds"),
                             (b.q, bounds.float(), b.scales[0], "bounds"), (b.q, bounds, b.scales[0][:2], "k_page_scale")):
        with pytest.raises(ValueError, match=message):
            decode.select(q, x, s)
    with pytest.raises(ValueError, match="selected"):
        run(decode, b, selected[:, :, :3])
    with pytest.raises(ValueError, match="selected"):
        run(decode, b, selected.long())
    with pytest.raises(RuntimeError, match="plan"):
        sparse.SelectedPagesDecode(torch.empty(1 << 20, device=cuda, dtype=torch.uint8)).select(b.q, bounds, b.scales[0])
    for codes, x, over, message in (
            (b.cache[0].float(), bounds, {}, "key_codes"), (b.cache[0], bounds[:3], {}, "bounds"),
            (b.cache[0], bounds, dict(page_ids=b.ids.long()), "page_ids"),
            (b.cache[0], bounds, dict(page_ids=b.ids, lengths=b.ids[:3]), "lengths")):
        with pytest.raises(ValueError, match=message):
            sparse.key_bounds(codes, x, **over)


def test_scores_are_the_headers(cuda):
    """Pages without tokens and scales of 0, both at once, and below it: the C header's formula
    as it stands, sum_d (max(q', 0) hi + min(q', 0) lo), for any bounds."""
    b = Batch(cuda, [], [3000, 1000], [0, 0], 2, 4)
    bounds = bounds_of(b, cuda)
    at = b.ids.long()
    for every, first in ((5, 1), (7, 2)):                 # some with a scale, some without
        bounds[at[first::every], :, 0], bounds[at[first::every], :, 1] = 127, -128
    b.scales[0][at[2::7]] = 0
    b.scales[0][at[3::11]] *= -1
    got = planned(b, cuda, 40, 0, 0, with_tail=False).select(b.q, bounds, b.scales[0]).cpu().numpy()
    q, low, high = b.q.double().cpu().numpy(), *bounds.cpu().numpy().astype(np.int64).transpose(2, 0, 1, 3)
    scale = b.scales[0].float().cpu().numpy()
    for i in range(2):
        ids = at[int(b.own_ptr[i]):int(b.own_ptr[i + 1])].cpu().numpy()
        for h in range(2):
            best = np.full(len(ids), -np.inf, np.float32)
            for row in q[i, 4 * h:4 * h + 4]:
                x = int(np.frexp(np.abs(row).max())[1])
                steps = np.clip(np.rint(np.ldexp(row, 7 - x)), -127, 127).astype(np.int64)
                total = (np.maximum(steps, 0) * high[ids, h] + np.minimum(steps, 0) * low[ids, h]).sum(1)
                best = np.maximum(best, np.float32(total) * scale[ids, h] * np.float32(2.0 ** (x - 7)))
            assert got[i, h].tolist() == sorted(np.argsort(-best, kind="stable")[:40])
