"""Attention over shared prefixes against float64 (tolerances: segment_helpers)."""

from __future__ import annotations

import pytest
import torch

from segment_helpers import Batch

pytestmark = pytest.mark.gpu

both_kinds = pytest.mark.parametrize("kind", [torch.int8, torch.float16])


def planned(batch, cuda, workspace_bytes=64 << 20, with_tail=True, **over):
    from pagegauge_amd import prefix

    decode = prefix.SharedPrefixDecode(torch.empty(workspace_bytes, device=cuda, dtype=torch.uint8))
    decode.plan([s[:2] for s in batch.segments], batch.prefix_ptr, batch.prefix_ids, batch.prefix_last,
                *batch.own_table(), *(batch.tail_table() if with_tail else ()),
                num_qo_heads=batch.hkv * batch.group, num_kv_heads=batch.hkv, kv_data_type=batch.kind, **over)
    return decode


def run(decode, batch, **over):
    a = dict(q=batch.q, kv_cache=batch.cache, k_page_scale=batch.scales[0], v_page_scale=batch.scales[1],
             exact_cache=batch.exact, value_center=batch.center, return_lse=True)
    a.update(over)
    return decode.run(**a)


def spread(count, low, high):
    return [low + (7 * i * i + 3 * i) % (high - low + 1) for i in range(count)]


# a token, inside a page, whole pages, past a tile, several items
@pytest.mark.parametrize("tokens", [1, 16, 17, 63, 1000, 5003])
@pytest.mark.parametrize("requests", [1, 2, 5, 9, 33])
@both_kinds
def test_lengths(cuda, tokens, requests, kind):
    print(f"prefix {tokens} x{requests} {kind}", flush=True)
    b = Batch(cuda, [(0, requests, tokens)], spread(requests, 0, 70), spread(requests, 0, 40), 2, 4, kind)
    b.check(*run(planned(b, cuda), b))


@pytest.mark.parametrize("kv_heads,group", [(8, 1), (5, 3), (1, 7), (4, 8), (2, 9), (2, 16), (16, 2)])
@pytest.mark.parametrize("requests", [3, 20])
@both_kinds
def test_head_layouts(cuda, kv_heads, group, requests, kind):
    print(f"prefix heads {kv_heads}x{group} x{requests} {kind}", flush=True)
    b = Batch(cuda, [(0, requests, 333)], spread(requests, 0, 50), spread(requests, 0, 20), kv_heads, group, kind)
    b.check(*run(planned(b, cuda), b))


@both_kinds
def test_nested_overlapping_empty_and_missing_prefixes(cuda, kind):
    segments = [(2, 9, 500), (0, 12, 33), (5, 9, 1), (9, 9, 40), (8, 12, 260), (3, 6, 0), (11, 12, 2000)]
    own = [0, 0, 17, 0, 300, 0, 0, 1, 0, 16, 0, 0, 0, 40]       # 12, 13: no prefix; 12: nothing at all
    tail = [0, 5, 0, 0, 16, 1, 0, 0, 0, 90, 0, 0, 0, 0]
    b = Batch(cuda, segments, own, tail, 2, 4, kind)
    out, lse = run(planned(b, cuda), b)
    b.check(out, lse)
    assert torch.equal(out[12], b.center[12].repeat_interleave(4, 0)) and bool((lse[12] == -torch.inf).all())


@both_kinds
def test_large_groups_and_long_prefixes(cuda, kind):
    print(f"prefix large {kind}", flush=True)
    b = Batch(cuda, [(0, 150, 2049), (20, 147, 3000)], spread(150, 0, 30), spread(150, 0, 9), 1, 4, kind)
    out, lse = run(planned(b, cuda), b)
    b.check(out, lse, requests=[0, 1, 19, 20, 21, 77, 146, 147, 149])


@pytest.mark.parametrize("longest,few", [(1000, True), (4000, False)])
@both_kinds
def test_many_requests(cuda, kind, longest, few):
    """More than 1024 (request, head) pairs, some without a join: with up to 16 partial rows
    joined a wave each, with more as few requests are."""
    own = spread(300, 0, 40)
    own[7], own[290] = longest, 0
    b = Batch(cuda, [(0, 280, 300), (100, 103, 77), (200, 260, 1200)], own, spread(300, 0, 18), 1, 4, kind)
    decode = planned(b, cuda)
    assert (decode._plan.max_slots <= 16) == few
    out, lse = run(decode, b)
    b.check(out, lse)
    again = run(decode, b, value_center=None)
    b.check(*again, center=False, requests=[0, 7, 101, 279, 280, 299])


def test_two_objects_on_two_streams(cuda):
    """Each with its own workspace, at the same time."""
    batches = [Batch(cuda, [(0, 40, 3000)], spread(40, 0, 200), spread(40, 0, 30), 2, 4, seed=s) for s in (1, 2)]
    decodes = [planned(b, cuda) for b in batches]
    want = [run(d, b) for d, b in zip(decodes, batches)]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (d, b) in enumerate(zip(decodes, batches)):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(d, b))
    torch.cuda.synchronize()
    for results, (out, lse) in zip(got, want):
        assert all(torch.equal(o, out) and torch.equal(l, lse) for o, l in results)


@both_kinds
def test_requests_without_any_prefix(cuda, kind):
    b = Batch(cuda, [], [5000, 0, 33], [100, 0, 16], 2, 4, kind)
    b.check(*run(planned(b, cuda), b), single_part=False)


@both_kinds
def test_no_own_pages_no_tail(cuda, kind):
    b = Batch(cuda, [(0, 6, 900)], [0] * 6, [0] * 6, 2, 4, kind)
    b.check(*run(planned(b, cuda, with_tail=False), b, exact_cache=None))


@both_kinds
def test_lengths_move_between_runs(cuda, kind):
    b = Batch(cuda, [(0, 5, 100), (2, 4, 48)], [20, 1, 0, 64, 5], [16, 3, 20, 1, 0], 2, 4, kind)
    decode = planned(b, cuda)
    for prefix_last, last, tail_last in (([1, 16], [16, 0, 0, 7, 1], [2, 0, 9, 16, 0]),
                                         ([0, 0], [0, 0, 0, 0, 0], [0, 0, 0, 0, 0])):
        b.prefix_last.copy_(torch.tensor(prefix_last))
        b.last.copy_(torch.tensor(last))
        b.tail_last.copy_(torch.tensor(tail_last))
        b.check(*run(decode, b))


@both_kinds
def test_rows_not_written_may_hold_anything(cuda, kind):
    """Infinities and NaN behind the last tokens, and in the scales of no page."""
    b = Batch(cuda, [(0, 40, 1005), (3, 5, 17)], spread(40, 0, 45), spread(40, 0, 35), 1, 4, kind)
    out, lse = run(planned(b, cuda), b)

    def spoil(pools, ptr, ids, last):
        for i in range(len(ptr) - 1):
            if ptr[i + 1] > ptr[i]:
                for p, bad in zip(pools, (float("nan"), float("inf"))):
                    p[ids[int(ptr[i + 1]) - 1], int(last[i]):] = bad

    if kind is torch.float16:
        spoil(b.cache, b.prefix_ptr, b.prefix_ids, b.prefix_last)
        spoil(b.cache, b.own_ptr, b.ids, b.last)
    else:
        used = torch.zeros(len(b.scales[0]), dtype=torch.bool)
        used[b.prefix_ids.cpu().long()] = True
        used[b.ids.cpu().long()] = True
        for s in b.scales:
            s[~used.to(cuda)] = float("nan")
    spoil(b.exact, b.tail_ptr, b.tail_ids, b.tail_last)
    got, got_lse = run(planned(b, cuda), b)
    assert torch.equal(got, out) and torch.equal(got_lse, lse)


@pytest.mark.parametrize("scale", [2.0 ** -13, 100.0])
def test_scales_of_any_size(cuda, scale):
    """Values far below and above 1 beside exact ones near 1."""
    b = Batch(cuda, [(0, 40, 700)], spread(40, 0, 30), spread(40, 0, 30), 1, 4, scale=scale)
    b.check(*run(planned(b, cuda), b))


def test_scales_that_differ_from_page_to_page(cuda):
    b = Batch(cuda, [(0, 40, 1500)], spread(40, 0, 30), [0] * 40, 1, 4)
    factor = 2.0 ** (torch.arange(len(b.scales[0]), device=cuda) % 13 - 8)[:, None]
    b.scales[1] = (b.scales[1].float() * factor).half()
    b.check(*run(planned(b, cuda), b))


@pytest.mark.parametrize("requests", [2, 10, 40])
def test_scales_of_either_sign(cuda, requests):
    """No writer makes them, but what they stand for is plain: code times scale."""
    b = Batch(cuda, [(0, requests, 900)], spread(requests, 0, 30), [0] * requests, 1, 4)
    sign = 1 - 2 * (torch.arange(len(b.scales[0]), device=cuda) % 3 == 1).half()[:, None]
    b.scales = [b.scales[0] * sign, b.scales[1] * sign.flip(0)]
    b.check(*run(planned(b, cuda), b))


@pytest.mark.parametrize("requests", [1, 3, 10, 30])
def test_small_values_beside_large_ones_without_weight(cuda, requests):
    """V's scales are of 2^-20, but for one page that no query attends to (its keys are far
    from all): the small values keep FP16's precision in every form.  A probability
    times its scale is 2^20 below what the largest scale could make it and 2^12 above the
    least FP16 value where that is put at 2^15: half a step is 2^-11 of it at most."""
    b = Batch(cuda, [(0, requests, 960)], [0] * requests, [0] * requests, 1, 4)
    b.q.abs_()
    b.q += 0.25
    b.scales[1].fill_(2.0 ** -20)
    far = int(b.prefix_ids[30])
    b.cache[0][far] = -128
    b.scales[0][far] = 4.0                       # scores of -128 * 4 * sum |q| sm: below -2000
    b.scales[1][far] = 1.0
    out, lse = run(planned(b, cuda), b, value_center=None)
    pools = [c[b.prefix_ids.long()].double().cpu() * s[b.prefix_ids.long()].double().cpu()[:, None, :, None]
             for c, s in zip(b.cache, b.scales)]
    k, v = (p.reshape(960, 128) for p in pools)
    scores = b.q.double().cpu() @ k.T * 128 ** -0.5
    weights = torch.softmax(scores, -1)
    want = weights @ v
    size = weights @ v.abs()                     # what the roundings of the terms are relative to
    # terms 2^-11 each, sums and exponents as in segment_helpers (scores below 2^6 here, but for
    # the far page's), then the output's half step: a subnormal's is 2^-25
    bound = size * (2.0 ** -11 + 2.0 ** -13) + 2.0 ** -25 + want.abs() * 2.0 ** -11
    assert bool(((out.double().cpu() - want).abs() <= bound).all())


@both_kinds
@pytest.mark.parametrize("requests", [1, 4, 30])
def test_infinite_scores(cuda, kind, requests):
    """Scores of -inf leave the others."""
    b = Batch(cuda, [(0, requests, 300)], [0] * requests, [20] * requests, 1, 4, kind)
    b.q.abs_()
    first = int(b.prefix_ids[0])
    decode = planned(b, cuda)
    if kind is torch.float16:
        b.cache[0][first, :, 0, 7] = float("-inf")
    else:
        b.cache[0][first] = -128
        b.scales[0][first] = float("inf")        # -128 * inf: -inf, for any q above 0
        b.q += 0.25
    out, lse = run(decode, b)
    b.prefix_ids, b.prefix_ptr[1] = b.prefix_ids[1:], int(b.prefix_ptr[1]) - 1     # as without that page
    b.check(out, lse)


@both_kinds
def test_scores_that_climb(cuda, kind):
    """The largest score is the last one, far above the others: every base moves."""
    b = Batch(cuda, [(0, 36, 800)], [20] * 36, [0] * 36, 1, 4, kind)
    if kind is torch.int8:
        climb = torch.linspace(0.002, 0.06, 50, device=cuda)
        b.scales[0][b.prefix_ids.long(), 0] = climb.half()
    else:
        climb = torch.linspace(0.1, 3.0, 50, device=cuda)
        b.cache[0][b.prefix_ids.long()] *= climb.half()[:, None, None, None]
    b.q *= 2
    b.check(*run(planned(b, cuda), b))


def test_a_spoiled_query_stays_in_its_row(cuda):
    b = Batch(cuda, [(0, 40, 300)], spread(40, 0, 30), spread(40, 0, 30), 2, 4)
    decode = planned(b, cuda)
    out, lse = run(decode, b)
    q = b.q.clone()
    q[7, 3] = float("nan")
    q[20, 0, 5] = float("inf")
    got, got_lse = run(decode, b, q=q)
    same = torch.ones(40, 8, dtype=torch.bool, device=cuda)
    same[7, 3] = same[20, 0] = False
    assert torch.equal(got[same], out[same]) and torch.equal(got_lse[same], lse[same])
    assert bool(got[7, 3].isnan().all())


@both_kinds
def test_given_outputs_strides_and_scale(cuda, kind):
    b = Batch(cuda, [(0, 3, 300)], [30, 0, 7], [20, 0, 3], 8, 4, kind)
    decode = planned(b, cuda)
    out, lse = run(decode, b, value_center=None)
    b.check(out, lse, center=False)
    wide = torch.empty(3, 48, 128, device=cuda, dtype=torch.float16)
    wide[:, :32] = b.q
    given, given_lse = torch.empty_like(out), torch.empty_like(lse)
    got = run(decode, b, q=wide[:, :32], value_center=None, out=given, lse=given_lse, return_lse=False)
    assert got is given and torch.equal(given, out) and torch.equal(given_lse, lse)
    scaled, scaled_lse = run(decode, b, sm_scale=0.5)
    b.check(scaled, scaled_lse, sm_scale=0.5)


@both_kinds
def test_runs_repeat_bit_by_bit_on_any_stream(cuda, kind):
    b = Batch(cuda, [(0, 50, 2000)], spread(50, 0, 90), spread(50, 0, 20), 2, 4, kind)
    decode = planned(b, cuda)
    out, lse = run(decode, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_lse = run(decode, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, out) and torch.equal(got_lse, lse)


def test_captured_runs_follow_their_inputs(cuda):
    cases = [Batch(cuda, [(0, 34, 500)], spread(34, 1, 40), spread(34, 1, 20), 2, 4, kind, seed=s)
             for s, kind in ((1, torch.int8), (2, torch.float16))]
    decodes = [planned(b, cuda, 32 << 20) for b in cases]
    graphs = []
    for decode, b in zip(decodes, cases):
        out, lse = run(decode, b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(decode, b, out=out, lse=lse)
        graphs.append((graph, out, lse))
    gen = torch.Generator().manual_seed(5)
    for _ in range(3):
        for (graph, out, lse), b in zip(graphs, cases):
            b.q.copy_(torch.randn(b.q.shape, generator=gen))
            b.last.clamp_(max=int(torch.randint(1, 17, (1,), generator=gen)))
            b.prefix_last.fill_(int(torch.randint(1, 17, (1,), generator=gen)))
            graph.replay()
        for (graph, out, lse), decode, b in zip(graphs, decodes, cases):
            torch.cuda.synchronize()
            want, want_lse = run(decode, b)
            assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_graphs_that_share_a_workspace(cuda):
    """Two captured runs of one object replayed in turn beside eager work."""
    b = Batch(cuda, [(0, 40, 700)], spread(40, 0, 60), spread(40, 0, 20), 2, 4)
    decode = planned(b, cuda)
    queries = [b.q, b.q.flip(0).contiguous()]
    want = [run(decode, b, q=q) for q in queries]
    outs = [(torch.empty_like(o), torch.empty_like(l)) for o, l in want]
    graphs = []
    for q, (out, lse) in zip(queries, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(decode, b, q=q, out=out, lse=lse)
    for _ in range(3):
        for graph, got, wanted in zip(graphs, outs, want):
            got[0].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], wanted[0]) and torch.equal(got[1], wanted[1])
        assert torch.equal(run(decode, b)[0], want[0][0])


def test_gradients_are_refused(cuda):
    b = Batch(cuda, [(0, 2, 40)], [20, 3], [5, 5], 2, 4)
    decode = planned(b, cuda)
    want = run(decode, b)
    follow = lambda t: t.clone().requires_grad_()  # noqa: E731
    for over in (dict(q=follow(b.q)), dict(value_center=follow(b.center)), dict(k_page_scale=follow(b.scales[0])),
                 dict(v_page_scale=follow(b.scales[1])), dict(exact_cache=(b.exact[0], follow(b.exact[1])))):
        with pytest.raises(ValueError, match="no gradient"):
            run(decode, b, **over)
        with torch.no_grad():
            assert torch.equal(run(decode, b, **over)[0], want[0])


def test_same_as_the_segmented_decode_over_whole_tables(cuda):
    """Each request's table with the prefix in front, by the operator that has no prefixes."""
    from pagegauge_amd.decode import PageGaugeSegmentedDecode

    b = Batch(cuda, [(0, 6, 512)], [16, 160, 32, 48, 16, 320], [20, 16, 3, 1, 40, 7], 8, 4)
    out, lse = run(planned(b, cuda), b)
    rows = [torch.cat((b.prefix_ids, b.ids[b.own_ptr[i]:b.own_ptr[i + 1]])) for i in range(6)]
    indptr = torch.tensor([0] + [len(r) for r in rows]).cumsum(0).int()
    whole = PageGaugeSegmentedDecode(torch.empty(64 << 20, device=cuda, dtype=torch.uint8))
    whole.plan(indptr, torch.cat(rows), torch.full((6,), 16, device=cuda, dtype=torch.int32), *b.tail_table())
    want = whole.run(b.q, b.cache, *b.scales, b.exact, b.center)
    # both are within their bounds of the same value: a step of FP16 and 2^-11 of the largest one
    assert bool(((out - want).abs().float() <= 2.0 ** -10 * want.abs().float() + 2.0 ** -10 * 2.6).all())


@both_kinds
def test_pools_past_2_to_the_31_bytes(cuda, kind):
    pages = (5 << 30) // (16 * 2 * 128 * (1 if kind is torch.int8 else 2)) // 2
    b = Batch(cuda, [(0, 34, 200)], spread(34, 0, 20), [0] * 34, 2, 4, kind)
    big = [torch.empty(pages, 16, 2, 128, dtype=kind, device=cuda) for _ in range(2)]
    shift = pages - len(b.cache[0])
    for x, c in zip(big, b.cache):
        x[shift:] = c
    decode = planned(b, cuda)
    out, lse = run(decode, b)
    if kind is torch.int8:
        scales = [torch.zeros(pages, 2, dtype=torch.float16, device=cuda) for _ in range(2)]
        for x, s in zip(scales, b.scales):
            x[shift:] = s
    else:
        scales = [None, None]
    b.prefix_ids += shift
    b.ids += shift
    got, got_lse = run(decode, b, kv_cache=big, k_page_scale=scales[0], v_page_scale=scales[1])
    assert torch.equal(got, out) and torch.equal(got_lse, lse)


def test_run_refuses(cuda):
    from pagegauge_amd import prefix

    b = Batch(cuda, [(0, 2, 40)], [20, 3], [5, 5], 2, 4)
    decode = planned(b, cuda)
    bad = [
        (dict(q=b.q.float()), "float16"), (dict(q=b.q[:1]), "does not match"),
        (dict(kv_cache=(b.cache[0], b.cache[1].half())), "int8"), (dict(k_page_scale=None), "need k_page_scale"),
        (dict(k_page_scale=b.scales[0][:3]), "k_page_scale"), (dict(exact_cache=None), "exact pages"),
        (dict(exact_cache=[e.float() for e in b.exact]), "exact_key"), (dict(value_center=b.center[:1]), "centers"),
        (dict(out=torch.empty(2, 8, 64, device=cuda).half()), "out must"), (dict(lse=b.q), "lse must"),
        (dict(q=b.q.clone().requires_grad_()), "no gradient"),
    ]
    for over, message in bad:
        with pytest.raises(ValueError, match=message):
            run(decode, b, **over)
    for sm_scale in (0.0, -1.0, float("nan"), 2.0 ** 100):
        with pytest.raises(RuntimeError, match="sm_scale"):
            run(decode, b, sm_scale=sm_scale)
    with pytest.raises(RuntimeError, match="plan"):
        run(prefix.SharedPrefixDecode(torch.empty(1 << 20, device=cuda, dtype=torch.uint8)), b)
    with pytest.raises(RuntimeError, match="workspace too small"):
        planned(b, cuda, 256)
    with pytest.raises(RuntimeError, match="range of the batch"):
        b.segments = [(0, 3, 40)]
        planned(b, cuda)
