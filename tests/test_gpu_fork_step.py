"""Requests forked from one prompt, as they are served: pages counted, shared and
taken, the fork's exact page copied, tokens appended by the serving tables' append,
bounds of completed pages, attention over the shared prompt and over selected pages,
requests that end, and the pool compacted under the others.

Every step's attention is held against float64 over the same pages (tolerances:
segment_helpers); what moves pages must change no bit of it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from segment_helpers import check_head, values

pytestmark = pytest.mark.gpu

HKV, GROUP, PROMPT = 2, 4, 37            # pages of the prompt; 5 tokens more lie in its exact page
CHILDREN, STEPS = 5, 40


def ints(values_, cuda):
    return torch.tensor(values_, dtype=torch.int32, device=cuda)


class Served:
    """One layer: a code pool, exact pages, bounds, and the requests' tables."""

    def __init__(self, cuda):
        from pagegauge_amd import pages, sparse
        from pagegauge_amd.decoder import rope_tables
        from pagegauge_amd.runtime import load_append_extension
        from pagegauge_amd.update import prefill_page_gauge, token_major_centers

        self.cuda, self.gen = cuda, torch.Generator().manual_seed(12)
        self.ext = load_append_extension()
        self.cos, self.sin = (t.to(cuda) for t in rope_tables(16 * PROMPT + 5 + STEPS + 18, 1e4))
        count = PROMPT + 40
        self.pool, self.exact_pool = pages.PagePool(count, device=cuda), pages.PagePool(12, device=cuda)
        self.codes = [torch.zeros(count, 16, HKV, 128, dtype=torch.int8, device=cuda) for _ in range(2)]
        self.scales = [torch.zeros(count, HKV, dtype=torch.float16, device=cuda) for _ in range(2)]
        self.exact = [torch.full((12, 16, HKV, 128), float("nan"), dtype=torch.float16, device=cuda) for _ in range(2)]
        self.bounds = sparse.allocate_bounds(count, HKV, cuda)

        tokens = 16 * PROMPT + 5
        k, v = (torch.randn(tokens, HKV, 128, generator=self.gen).half().to(cuda) for _ in range(2))
        key_center, value_center = token_major_centers(k, v)
        # the prompt's pages are not the pool's first ones: an earlier request holds those
        self.earlier = self.pool.take(20)
        self.prompt = self.pool.take(PROMPT)
        at = slice(int(self.prompt[0]), int(self.prompt[0]) + PROMPT)
        prefill_page_gauge(k[:16 * PROMPT], v[:16 * PROMPT], key_center, value_center, self.codes[0][at],
                           self.codes[1][at], self.scales[0][at], self.scales[1][at])
        sparse.key_bounds(self.codes[0], self.bounds, page_ids=self.prompt)
        parent = self.exact_pool.take(1)
        for e, rows, center in zip(self.exact, (k, v), (key_center, value_center)):
            e[parent.long(), :5] = (rows[16 * PROMPT:].float() - center.float()).half()

        # the fork: each child a user of the prompt's pages, with a copy of the exact one
        self.pool.share(self.prompt, CHILDREN - 1)
        self.exact_ids = torch.cat((parent, self.exact_pool.take(CHILDREN - 1)))
        pages.copy_pages(self.exact, parent.expand(CHILDREN - 1).contiguous(), self.exact_ids[1:])
        self.centers = [c.expand(CHILDREN, HKV, 128).contiguous() for c in (key_center, value_center)]
        self.requests = CHILDREN
        self.own = [[] for _ in range(CHILDREN)]             # code pages completed since the fork
        self.next_ids = self.pool.take(CHILDREN)             # where the current page will be held
        self.position = 16 * PROMPT + 5

    def append(self):
        from pagegauge_amd import sparse

        n = self.requests
        q = torch.randn(n, HKV * GROUP, 128, generator=self.gen).half().to(self.cuda)
        k, v = (torch.randn(n, HKV, 128, generator=self.gen).half().to(self.cuda) for _ in range(2))
        rotated = torch.empty_like(q)
        positions = ints([self.position] * n, self.cuda)
        self.ext.rope_append_page_gauge_slots(
            q, k, v, self.cos, self.sin, positions, self.exact_ids, self.next_ids, *self.centers, rotated,
            *self.exact, *self.codes, *self.scales)
        self.position += 1
        if self.position % 16 == 0:                          # the page is history now
            sparse.key_bounds(self.codes[0], self.bounds, page_ids=self.next_ids)
            for own, page in zip(self.own, self.next_ids.tolist()):
                own.append(page)
            self.next_ids = self.pool.take(n)
        return rotated

    def plan(self, picked):
        """Both operators over the tables as they are now."""
        from pagegauge_amd import prefix, sparse

        n, tail = self.requests, self.position % 16
        own = [len(o) for o in self.own]
        own_ptr = torch.tensor([0] + own).cumsum(0).int()
        self.own_ids = ints([p for o in self.own for p in o] + [0], self.cuda)
        self.whole = torch.cat([torch.cat((self.prompt, ints(o, self.cuda))) for o in self.own])
        full = ints([16] * n, self.cuda)
        tail_ptr = torch.arange(n + 1).int() * (tail > 0)
        tail_table = tail_ptr, self.exact_ids, ints([tail] * n, self.cuda)
        shared = prefix.SharedPrefixDecode(torch.empty(8 << 20, device=self.cuda, dtype=torch.uint8))
        shared.plan([(0, n)], [0, PROMPT], self.prompt, ints([16], self.cuda), own_ptr, self.own_ids, full, *tail_table,
                    num_qo_heads=HKV * GROUP, num_kv_heads=HKV)
        part = sparse.SelectedPagesDecode(torch.empty(8 << 20, device=self.cuda, dtype=torch.uint8))
        part.plan(own_ptr + PROMPT * torch.arange(n + 1).int(), self.whole, full, *tail_table, pages=picked,
                  num_qo_heads=HKV * GROUP, num_kv_heads=HKV)
        return shared, part

    def run_shared(self, decode, q):
        return decode.run(q, self.codes, *self.scales, self.exact, value_center=self.centers[1], return_lse=True)

    def run_part(self, decode, q):
        selected = decode.select(q, self.bounds, self.scales[0])
        return (selected, *decode.run(q, self.codes, *self.scales, selected, self.exact,
                                      value_center=self.centers[1], return_lse=True))

    def check(self, q, out, lse, selected=None):
        pools = [values(c, s) for c, s in zip(self.codes, self.scales)]
        tail = [values(e, None)[self.exact_ids.cpu().numpy(), :self.position % 16] for e in self.exact]
        out, lse, q = (t.double().cpu().numpy() for t in (out, lse, q))
        center = self.centers[1].cpu().numpy()
        for b in range(self.requests):
            ids = np.array(self.prompt.tolist() + self.own[b])
            for h in range(HKV):
                at = ids if selected is None else ids[[p for p in selected[b, h].tolist() if p >= 0]]
                k, v = (np.concatenate((p[at, :, h].reshape(-1, 128), t[b, :, h])) for p, t in zip(pools, tail))
                rows = slice(GROUP * h, GROUP * (h + 1))
                check_head(out[b, rows], lse[b, rows], q[b, rows], k, v, center[b, h], 128 ** -0.5, True)


def test_forked_requests_step_by_step(cuda):
    from pagegauge_amd import pages

    s = Served(cuda)
    for step in range(STEPS):
        q = s.append()
        if step % 7 and step != STEPS - 1:
            continue
        shared, part = s.plan(picked=9)
        out, lse = s.run_shared(shared, q)
        s.check(q, out, lse)
        selected, out, lse = s.run_part(part, q)
        s.check(q, out, lse, selected)
        _, everything = s.plan(picked=PROMPT + 9)            # all pages taken: the same attention
        s.check(q, *s.run_part(everything, q)[1:])

    # counts: the prompt's pages have a user per child, own pages one
    refs = s.pool.refs.tolist()
    assert [refs[p] for p in s.prompt.tolist()] == [CHILDREN] * PROMPT
    assert [refs[p] for o in s.own for p in o] == [1] * sum(map(len, s.own))

    # two children and the earlier request end
    for b in (3, 1):
        s.pool.release(torch.cat((s.prompt, ints(s.own.pop(b), cuda), s.next_ids[b:b + 1])))
        s.exact_pool.release(s.exact_ids[b:b + 1])
        keep = [i for i in range(s.requests) if i != b]
        s.exact_ids, s.next_ids = s.exact_ids[keep], s.next_ids[keep]
        s.centers = [c[keep] for c in s.centers]
        s.requests -= 1
    s.pool.release(s.earlier)
    q = s.append()
    shared, part = s.plan(picked=9)
    before = *s.run_shared(shared, q), *s.run_part(part, q)
    s.check(q, *before[:2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = *s.run_shared(shared, q), *s.run_part(part, q)

    # the pool compacted, tables rewritten in place: not a bit of the attention changes,
    # called again or replayed
    moves = s.pool.stage_compaction()
    pages.copy_pages((*s.codes, *s.scales, s.bounds), moves.source, moves.target)
    live = int(moves.live)
    assert int((moves.source >= 0).sum()) > 0
    for table in (s.prompt, s.own_ids[:-1], s.whole, s.next_ids):
        pages.rewrite_ids(table, moves.remap, out=table)
    s.own = [pages.rewrite_ids(ints(o, cuda), moves.remap).tolist() for o in s.own]
    s.pool.commit_compaction(moves)
    for plane in (*s.codes, *s.scales, s.bounds):
        plane[live:] = 111                                   # nothing is read there any more
    after = *s.run_shared(shared, q), *s.run_part(part, q)
    assert all(torch.equal(x, y) for x, y in zip(before, after))
    for _ in range(2):
        for t in captured:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(before, captured))
    assert bool((s.pool.refs[:live] > 0).all()) and not bool(s.pool.refs[live:].any())

    # and the step goes on, into pages freshly taken
    for _ in range(17):
        q = s.append()
    shared, part = s.plan(picked=9)
    s.check(q, *s.run_shared(shared, q))
    selected, out, lse = s.run_part(part, q)
    s.check(q, out, lse, selected)
