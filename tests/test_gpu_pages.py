"""Pages copied, counted, handed out and moved, against lists."""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def filled(cuda, shape, dtype, gen):
    x = torch.randint(-120, 120, shape, generator=gen)
    return (x if dtype != torch.uint8 else x.abs()).to(dtype).to(cuda)


# bytes of a page: 1, 2, 6, 33, 12, 16, 24, 4112, 32768
@pytest.mark.parametrize("page,dtype", [
    ((), torch.int8), ((1,), torch.float16), ((3,), torch.float16), ((33,), torch.uint8), ((3,), torch.int32),
    ((8,), torch.float16), ((3, 2, 4), torch.uint8), ((257, 8), torch.float16), ((16, 8, 128), torch.float16)])
@pytest.mark.parametrize("layers", [None, 1, 3])
def test_copies(cuda, page, dtype, layers):
    from pagegauge_amd import pages

    print(f"copy {page} {dtype} {layers}", flush=True)
    gen = torch.Generator().manual_seed(2)
    shape = (71, *page) if layers is None else (layers, 71, *page)
    plane = filled(cuda, shape, dtype, gen)
    order = torch.randperm(71, generator=gen).tolist()
    target = order[:40] + [-1, 71, 2 ** 31 - 1, order[69], -5]
    source = [order[50 + i % 13] for i in range(40)] + [order[66], order[66], order[66], 71, order[66]]
    want = plane.clone()
    for s, t in zip(source[:40], target):
        if layers is None:
            want[t] = plane[s]
        else:
            want[:, t] = plane[:, s]
    pages.copy_pages([plane], ints(source, cuda), ints(target, cuda), page_dim=0 if layers is None else 1)
    assert torch.equal(plane, want)


def test_copies_of_many_planes_at_odd_places(cuda):
    """Layers of a pool as planes of their own, views that start anywhere, page strides
    longer than a page, several launches."""
    from pagegauge_amd import pages

    gen = torch.Generator().manual_seed(3)
    store = filled(cuda, (40, 30, 50), torch.uint8, gen)
    planes = [store[i, :, 3:3 + 1 + i % 17] for i in range(40)]
    interleaved = filled(cuda, (30, 4, 7), torch.int8, gen).transpose(0, 1)      # layers within pages
    planes_before, before = store.clone(), interleaved.clone()
    source, target = ints([3, 4, 5, 3], cuda), ints([10, 29, 0, 11], cuda)
    pages.copy_pages(planes, source, target)
    pages.copy_pages([interleaved], source, target, page_dim=1)
    for s, t in zip(source.tolist(), target.tolist()):
        for i in range(40):
            planes_before[i, t, 3:4 + i % 17] = planes_before[i, s, 3:4 + i % 17]
        before[:, t] = before[:, s]
    assert torch.equal(store, planes_before) and torch.equal(interleaved, before)


def test_copies_past_2_to_the_32_bytes(cuda):
    from pagegauge_amd import pages

    plane = torch.zeros(300_000, 16384, dtype=torch.uint8, device=cuda)
    plane[299_999] = torch.arange(16384, device=cuda) % 251
    pages.copy_pages([plane], ints([299_999, 299_999], cuda), ints([299_990, 1], cuda))
    assert torch.equal(plane[299_990], plane[299_999]) and torch.equal(plane[1], plane[299_999])
    assert int(plane[2].sum()) == int(plane[299_991].sum()) == 0


def test_copies_of_nothing(cuda):
    from pagegauge_amd import pages

    none = ints([], cuda)
    plane = torch.ones(4, 8, device=cuda)
    pages.copy_pages([plane], none, none)
    pages.copy_pages([torch.ones(0, 8, device=cuda)], ints([0], cuda), ints([1], cuda))
    pages.copy_pages([torch.ones(4, 0, device=cuda), plane], ints([-1], cuda), ints([1], cuda))
    assert bool((plane == 1).all())
    plane[2] = 5
    pages.copy_pages((p for p in (plane,)), ints([2], cuda), ints([0], cuda))      # any iterable
    assert bool((plane[0] == 5).all())


def test_counts(cuda):
    from pagegauge_amd import pages

    rng = random.Random(4)
    pool = pages.PagePool(1000, device=cuda)
    want = [0] * 1000
    for _ in range(6):
        ids = [rng.choice([-1, -7, 1000, 2 ** 31 - 1, rng.randrange(40), rng.randrange(1000)]) for _ in range(3000)]
        users = rng.randint(1, 3)
        pool.share(ints(ids, cuda), users)
        for i in ids:
            if 0 <= i < 1000:
                want[i] += users
        assert pool.refs.tolist() == want
        ids = [rng.choice([-1, 1000, rng.randrange(40), rng.randrange(1000)]) for _ in range(4000)]
        users = rng.randint(1, 4)
        pool.release(ints(ids, cuda), users)
        for i in ids:
            if 0 <= i < 1000:
                want[i] = max(want[i] - users, 0)
        assert pool.refs.tolist() == want


SIZES = [1, 2, 15, 16, 17, 1000, 16384, 16385, 50001]


@pytest.mark.parametrize("pages_in_pool", SIZES)
def test_take(cuda, pages_in_pool):
    from pagegauge_amd import pages

    print(f"take {pages_in_pool}", flush=True)
    rng = random.Random(pages_in_pool)
    for live in (0.0, 0.5, 0.97, 1.0):
        pool = pages.PagePool(pages_in_pool, device=cuda)
        refs = [int(rng.random() < live) * rng.randint(1, 5) for _ in range(pages_in_pool)]
        for count in (1, 7, pages_in_pool // 3, pages_in_pool + 3):
            pool.refs.copy_(ints(refs, cuda))
            free = [p for p in range(pages_in_pool) if not refs[p]][:count]
            got = pool.take(count)
            assert got.tolist() == free + [-1] * (count - len(free))
            want = list(refs)
            for p in free:
                want[p] = 1
            assert pool.refs.tolist() == want
    assert pool.take(0).numel() == 0


def expected_moves(refs):
    live = sum(r > 0 for r in refs)
    holes = [p for p in range(live) if refs[p] <= 0]
    movers = [p for p in range(live, len(refs)) if refs[p] > 0]
    remap = [p if r > 0 else -1 for p, r in enumerate(refs)]
    for s, t in zip(movers, holes):
        remap[s] = t
    return live, movers, holes, remap


@pytest.mark.parametrize("pages_in_pool", [0] + SIZES)
def test_compaction(cuda, pages_in_pool):
    from pagegauge_amd import pages

    print(f"compact {pages_in_pool}", flush=True)
    rng = random.Random(pages_in_pool)
    pool = pages.PagePool(pages_in_pool, device=cuda)
    moves = None
    for live_part in (0.0, 0.03, 0.5, 0.9, 1.0):
        refs = [int(rng.random() < live_part) * rng.randint(1, 5) for _ in range(pages_in_pool)]
        pool.refs.copy_(ints(refs, cuda))
        moves = pool.stage_compaction(out=moves)
        live, movers, holes, remap = expected_moves(refs)
        pad = [-1] * (pages_in_pool // 2 - len(movers))
        assert moves.live.tolist() == [live] and moves.remap.tolist() == remap
        assert moves.source.tolist() == movers + pad and moves.target.tolist() == holes + pad
        assert pool.refs.tolist() == refs
        plane = torch.arange(pages_in_pool, device=cuda)
        pages.copy_pages([plane], moves.source, moves.target)
        used = [p for p in range(pages_in_pool) if refs[p]]
        table = ints(used + [-1, pages_in_pool, -9], cuda)
        new = pages.rewrite_ids(table, moves.remap)
        assert new.tolist()[-3:] == [-1, pages_in_pool, -9]
        assert sorted(new.tolist()[:-3]) == list(range(live))
        assert plane[new[:-3].long()].tolist() == used             # each page's content went with it
        assert pages.rewrite_ids(table, moves.remap, out=table) is table and torch.equal(table, new)
        pool.commit_compaction(moves)
        want = [0] * pages_in_pool
        for p in used:
            want[remap[p]] = refs[p]
        assert pool.refs.tolist() == want
        pool.commit_compaction(moves)                              # once more: nothing is left to move
        assert pool.refs.tolist() == want


def test_captured_calls_follow_the_pool(cuda):
    from pagegauge_amd import pages

    pool = pages.PagePool(300, device=cuda)
    plane = torch.arange(300, device=cuda)
    moves, taken = pool.stage_compaction(), pool.take(5)
    freed, table = ints([-1] * 40, cuda), ints([-1] * 40, cuda)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.release(freed)
        pool.stage_compaction(out=moves)
        pages.copy_pages([plane], moves.source, moves.target)
        pages.rewrite_ids(table, moves.remap, out=table)
        pool.commit_compaction(moves)
        pool.take(5, out=taken)
    rng = random.Random(6)
    for _ in range(4):
        refs = [rng.choice([0, 1, 2]) for _ in range(300)]
        ids = rng.sample(range(300), 40)
        left = [max(r - (p in ids), 0) for p, r in enumerate(refs)]
        used = [p for p in range(300) if left[p]][:40]
        pool.refs.copy_(ints(refs, cuda))
        freed.copy_(ints(ids, cuda))
        table.copy_(ints(used, cuda))
        plane.copy_(torch.arange(300))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        live, _, _, remap = expected_moves(left)
        assert table.tolist() == [remap[p] for p in used] and plane[table.long()].tolist() == used
        assert taken.tolist() == list(range(live, live + 5))
        assert int((pool.refs > 0).sum()) == live + 5


def test_refuses(cuda):
    from pagegauge_amd import pages

    plane, one = torch.zeros(4, 8, device=cuda), ints([1], cuda)
    for planes, source, target, over, message in (
            ([plane], one.long(), one.long(), {}, "int32"), ([plane], one, ints([1, 2], cuda), {}, "one id per copy"),
            ([], one, one, {}, "no planes"), (plane, one, one, {}, "sequence of tensors"), ([plane, plane[:3]], one, one, {}, "same number of pages"),
            ([plane[:, ::2]], one, one, {}, "contiguous"), ([plane[:1].expand(4, 8)], one, one, {}, "overlap"),
            ([plane[None].expand(2, 4, 8)], one, one, dict(page_dim=1), "overlap"),
            ([plane], one, one, dict(page_dim=2), "page_dim"), ([plane.cpu()], one, one, {}, "device"),
            ([plane[0, 0]], one, one, {}, "dimension"),
            ([plane.clone().requires_grad_()], one, one, {}, "no gradient")):
        with pytest.raises(ValueError, match=message):
            pages.copy_pages(planes, source, target, **over)
    pool = pages.PagePool(4, device=cuda)
    other = pages.PagePool(6, device=cuda)
    for call, message in ((lambda: pool.share(one, 0), "positive"), (lambda: pool.release(one, -1), "positive"),
                          (lambda: pool.share(one.long()), "int32"), (lambda: pool.share(one.cpu()), "device"),
                          (lambda: pool.take(-1), "nonnegative"), (lambda: pool.take(2, out=one), "int32"),
                          (lambda: pool.stage_compaction(out=other.stage_compaction()), "of this pool"),
                          (lambda: pages.rewrite_ids(one.long(), one), "int32"),
                          (lambda: pages.rewrite_ids(one, one, out=ints([1, 2], cuda)), "int32"),
                          (lambda: pages.PagePool(-1), "2\\^31")):
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(RuntimeError, match="more moves"):
        pool.commit_compaction(pages.PagePool(20, device=cuda).stage_compaction())


@pytest.mark.parametrize("users", [1, 2 ** 20, 2 ** 30, 2 ** 31 - 1])
def test_counts_stay_at_the_largest(cuda, users):
    """A count past int32 stays at 2^31 - 1 for good: the page is never handed out."""
    from pagegauge_amd import pages

    most = 2 ** 31 - 1
    pool = pages.PagePool(8, device=cuda)
    pool.refs.copy_(ints([0, most - 1, most, most - users, 5, 1, 1, 1], cuda))
    ids = [0, 1, 2, 3, 3, -1, 8] + [4] * 5000
    pool.share(ints(ids, cuda), users)
    want = [min(users, most), most, most, most, min(5 + 5000 * users, most), 1, 1, 1]
    assert pool.refs.tolist() == want
    pool.release(ints([1, 2, 3, 3, 0], cuda), users)
    want[0] = most if users == most else 0
    assert pool.refs.tolist() == want
    assert pool.take(8).tolist() == ([-1] if users == most else [0]) + [-1] * 7
