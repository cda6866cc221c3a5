"""The operators as a decode step uses them: prompts rotated and held in 4 bits,
then token by token rotation and append, attention over history and exact
pages, logits shaped and the next token picked."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int4_helpers import attention, unpack

pytestmark = pytest.mark.gpu

HKV, GROUP, VOCAB, RING = 2, 4, 997, 2
HQ = HKV * GROUP


class Served:
    """Requests of their own lengths over one pool; the page a request is in
    and the one before are exact, older pages 4-bit."""

    def __init__(self, cuda, prompts, steps):
        from pagegauge_amd import int4, rotary

        gen = torch.Generator().manual_seed(len(prompts))
        half = lambda *s: torch.randn(*s, generator=gen).half().to(cuda)  # noqa: E731
        self.device, self.batch = cuda, len(prompts)
        self.length = list(prompts)
        self.rotary = rotary.RotaryEmbedding(128, 64, layout="interleaved", scaling="by_parts",
                                             factor=4.0, original_context=64)
        self.embed = half(VOCAB, (HQ + 2 * HKV) * 128)
        self.head = half(HQ * 128, VOCAB) * 0.05
        pages = [-(-(n + steps) // 16) for n in prompts]
        self.codes, self.scales = int4.allocate_pages(sum(pages) + 1, HKV, cuda)
        ids = torch.randperm(sum(pages) + 1, generator=gen)[:sum(pages)].int()
        self.pages = ids.split(pages)
        self.exact = [half(self.batch * RING, 16, HKV, 128) for _ in range(2)]
        self.centers = [torch.zeros(self.batch, HKV, 128, device=cuda, dtype=torch.float16)
                        for _ in range(2)]
        self.history = torch.zeros(self.batch, max(prompts) + steps, device=cuda, dtype=torch.int64)
        self.tokens = torch.zeros(self.batch, device=cuda, dtype=torch.int64)
        for b, n in enumerate(prompts):
            tokens = torch.randint(0, VOCAB, (n + 1,), generator=gen).to(cuda)
            self.history[b, :n] = tokens[:n]
            self.tokens[b] = tokens[n]
            qkv = self.embed[tokens[:n]]
            _, key = self.rotary.rotate(qkv[:, :HQ * 128].view(n, HQ, 128),
                                        qkv[:, HQ * 128:(HQ + HKV) * 128].view(n, HKV, 128),
                                        torch.arange(n, device=cuda))
            value = qkv[:, (HQ + HKV) * 128:].view(n, HKV, 128)
            for c, x in zip(self.centers, (key, value)):
                c[b] = x.float().mean(0).half()
            count = -(-n // 16)
            # the last pages are exact as well, in slot page % RING
            slots = [b * RING + p % RING if p >= count - RING else -1 for p in range(count)]
            int4.quantize_pages(key, value, self.codes, self.scales,
                                page_ids=self.pages[b][:count].to(cuda),
                                key_center=self.centers[0][b], value_center=self.centers[1][b],
                                exact_page_ids=torch.tensor(slots, device=cuda, dtype=torch.int32),
                                exact_key=self.exact[0], exact_value=self.exact[1])
        self.prompt_lengths = torch.tensor(prompts, device=cuda, dtype=torch.int32)
        self.positions = torch.zeros(self.batch, device=cuda, dtype=torch.int32)
        self.exact_ids, self.code_ids = torch.zeros_like(self.positions), torch.zeros_like(self.positions)
        self.counts = torch.zeros_like(self.positions)
        self.old_last = torch.full_like(self.positions, 16)
        self.tail_last = torch.zeros_like(self.positions)
        self.penalty = torch.full((self.batch,), 1.5, device=cuda)
        self.allowed = torch.full((self.batch, -(-VOCAB // 32)), -1, device=cuda, dtype=torch.int32)
        self.allowed[:, 3] = 0
        self.decode = int4.Int4PagedDecode(torch.empty(16 << 20, device=cuda, dtype=torch.uint8))
        self.rotated = torch.empty(self.batch, HQ, 128, device=cuda, dtype=torch.float16)
        self.out = torch.empty_like(self.rotated)
        self.lse = torch.empty(self.batch, HQ, device=cuda)
        self.logits = torch.empty(self.batch, VOCAB, device=cuda)
        self.shaped = torch.empty_like(self.logits)
        self.signature = None

    def prepare(self):
        """The step's tables for the tokens at ``length``; True when the page
        structure is a new one."""
        at = self.length
        current = [n // 16 for n in at]
        first = [max(0, p - RING + 1) for p in current]
        self.old = [self.pages[b][:first[b]] for b in range(self.batch)]
        self.tail = [torch.tensor([b * RING + p % RING for p in range(first[b], current[b] + 1)],
                                  dtype=torch.int32) for b in range(self.batch)]
        fill = lambda t, x: t.copy_(torch.tensor(x, dtype=torch.int32))  # noqa: E731
        fill(self.positions, at)
        fill(self.exact_ids, [b * RING + current[b] % RING for b in range(self.batch)])
        fill(self.code_ids, [int(self.pages[b][current[b]]) for b in range(self.batch)])
        fill(self.counts, [n + 1 for n in at])
        fill(self.tail_last, [n % 16 + 1 for n in at])
        for b, n in enumerate(at):
            self.history[b, n] = self.tokens[b]
        signature = tuple(current)
        if signature == self.signature:
            return False
        self.signature = signature
        tables = []
        for parts in (self.old, self.tail):
            indptr = torch.tensor([0] + list(np.cumsum([len(p) for p in parts])), dtype=torch.int32)
            tables.append((indptr, torch.cat(parts).to(self.device)))
        self.decode.plan(*tables[0], self.old_last, *tables[1], self.tail_last, num_qo_heads=HQ,
                         num_kv_heads=HKV)
        return True

    def step(self):
        from pagegauge_amd import int4
        from pagegauge_amd.decoder import argmax_rows
        from pagegauge_amd.logits import shape_logits

        b = self.batch
        qkv = self.embed[self.tokens]
        int4.rope_append(self.rotary, qkv[:, :HQ * 128].view(b, HQ, 128),
                         qkv[:, HQ * 128:(HQ + HKV) * 128].view(b, HKV, 128),
                         qkv[:, (HQ + HKV) * 128:].view(b, HKV, 128), self.positions, self.exact_ids,
                         self.code_ids, *self.centers, self.rotated, *self.exact, self.codes, self.scales)
        self.decode.run(self.rotated, self.codes, self.scales, self.exact, value_center=self.centers[1],
                        out=self.out, lse=self.lse)
        torch.mm(self.out.view(b, HQ * 128).float(), self.head.float(), out=self.logits)
        shape_logits(self.logits, self.shaped, history=self.history, history_lengths=self.counts,
                     prompt_lengths=self.prompt_lengths, repetition=self.penalty, presence=self.penalty,
                     allowed=self.allowed)
        argmax_rows(self.shaped, self.tokens)

    def advance(self):
        self.length = [n + 1 for n in self.length]

    def check(self):
        """Attention of the step just made, over what the cache now holds."""
        (kc, ks), (vc, vs) = unpack(self.codes, self.scales)
        pools = [(kc * ks.astype(np.float64)[..., None], vc * vs.astype(np.float64)[..., None]),
                 tuple(t.double().cpu().numpy() for t in self.exact)]
        for b in range(self.batch):
            parts = [], []
            for ids, pool, tokens in ((self.old[b], pools[0], 16 * len(self.old[b])),
                                      (self.tail[b], pools[1], self.length[b] + 1 - 16 * len(self.old[b]))):
                for out, x in zip(parts, pool):
                    out.append(x[ids.numpy()].reshape(-1, HKV, 128)[:tokens])
            k, v = (np.concatenate(p) for p in parts)
            assert len(k) == self.length[b] + 1
            want, lse, bound, lse_bound = attention(self.rotated[b].cpu().numpy(), k, v,
                                                    self.centers[1][b].cpu().numpy(), 128 ** -0.5)
            got = self.out[b].double().cpu().numpy()
            allowed = (np.abs(want) + bound[:, None]) * 2.0 ** -11 + bound[:, None] + 2.0 ** -24
            assert (np.abs(got - want) <= allowed).all()
        assert (self.tokens < VOCAB).all() and not ((self.tokens >= 96) & (self.tokens < 128)).any()
        assert torch.equal(self.tokens, self.shaped.argmax(-1))


def test_decode_steps(cuda):
    """Steps over page ends, prompts that end inside and at the end of a page."""
    s = Served(cuda, [5, 31, 200, 64], 40)
    for _ in range(40):
        s.prepare()
        s.step()
        s.check()
        s.advance()


def test_captured_steps_equal_eager_ones(cuda):
    """The steps of one page window as one graph, replayed with eager work
    between; the same tokens and caches as the eager steps."""
    eager, graphed = (Served(cuda, [16, 160], 16) for _ in range(2))
    for _ in range(15):
        eager.prepare()
        eager.step()
        eager.advance()
    graphed.prepare()
    keep = [t.clone() for t in (graphed.tokens, *graphed.exact, graphed.codes, graphed.scales)]
    graphed.step()                                      # warm-up
    for t, was in zip((graphed.tokens, *graphed.exact, graphed.codes, graphed.scales), keep):
        t.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.step()
    for _ in range(15):
        assert not graphed.prepare()
        graph.replay()
        torch.cuda.synchronize()
        graphed.check()
        graphed.advance()
    for name in ("tokens", "history", "codes", "scales", "out", "lse", "shaped"):
        assert torch.equal(getattr(eager, name), getattr(graphed, name)), name
    assert all(torch.equal(a, b) for a, b in zip(eager.exact, graphed.exact))


def test_serving_tables(cuda):
    """The tables of ``serving.decode_tables`` drive the step: exact sink, suffix
    and ring pages, history in 4 bits, pages that a step completed read back."""
    from pagegauge_amd import int4, rotary, serving as sv

    gen = torch.Generator().manual_seed(11)
    half = lambda *s: torch.randn(*s, generator=gen).half().to(cuda)  # noqa: E731
    pol = sv.Policy(prefix_pages=1, suffix_pages=2, tail_pages=2)
    ledger, rope = sv.Ledger(2, pol), rotary.RotaryEmbedding(128)
    codes, scales = int4.allocate_pages(64, HKV, cuda)
    exact = [half(2 * pol.storage_pages, 16, HKV, 128) for _ in range(2)]
    centers = [torch.zeros(2, HKV, 128, device=cuda, dtype=torch.float16) for _ in range(2)]
    free = torch.randperm(64, generator=gen).tolist()
    leases, tables = [], []
    for prompt in (200, 133):
        count = -(-prompt // 16)
        tables.append([free.pop() for _ in range(count)])
        lease = ledger.admit(f"request {prompt}", prompt, tables[-1], ready=True)
        leases.append(lease)
        key, value = half(prompt, HKV, 128), half(prompt, HKV, 128)
        for c, x in zip(centers, (key, value)):
            c[lease.slot] = x.float().mean(0).half()
        pages = sv.partition(prompt, prompt, pol)["exact"]
        slots = [sv.exact_slot(p, prompt, lease.slot, pol) if p in pages else -1 for p in range(count)]
        int4.quantize_pages(key, value, codes, scales,
                            page_ids=torch.tensor(tables[-1], device=cuda, dtype=torch.int32),
                            key_center=centers[0][lease.slot], value_center=centers[1][lease.slot],
                            exact_page_ids=torch.tensor(slots, device=cuda, dtype=torch.int32),
                            exact_key=exact[0], exact_value=exact[1])
    decode = int4.Int4PagedDecode(torch.empty(16 << 20, device=cuda, dtype=torch.uint8))
    completed, read_back = set(), set()
    for _ in range(70):
        scheduled = []
        for lease, table in zip(leases, tables):
            at = ledger.view(lease).current_tokens
            if at % 16 == 0:
                table.append(free.pop())
            scheduled.append((lease, at, table))
        batch = ledger.stage_decode(scheduled)
        t = sv.decode_tables(batch, pol, device=cuda)
        read_back |= completed & set(t.old_indices.tolist())
        completed |= {table[at // 16] for _, at, table in scheduled if at % 16 == 15}
        kc, vc = (c[t.request_slots.long()].contiguous() for c in centers)
        rotated = torch.empty(2, HQ, 128, device=cuda, dtype=torch.float16)
        int4.rope_append(rope, half(2, HQ, 128), half(2, HKV, 128), half(2, HKV, 128), t.positions,
                         t.exact_page_ids, t.code_page_ids, kc, vc, rotated, *exact, codes, scales)
        decode.plan(t.old_indptr, t.old_indices, t.old_last_page_len, t.exact_indptr,
                    t.exact_indices, t.exact_last_page_len, num_qo_heads=HQ, num_kv_heads=HKV)
        out = decode.run(rotated, codes, scales, exact, value_center=vc)
        (kq, ks), (vq, vs) = unpack(codes, scales)
        pools = [(kq * ks.astype(np.float64)[..., None], vq * vs.astype(np.float64)[..., None]),
                 tuple(x.double().cpu().numpy() for x in exact)]
        for b, (_, at, _) in enumerate(scheduled):
            old = t.old_indices[t.old_indptr[b]:t.old_indptr[b + 1]].cpu().numpy()
            new = t.exact_indices[t.exact_indptr[b]:t.exact_indptr[b + 1]].cpu().numpy()
            k, v = (np.concatenate([pools[0][i][old], pools[1][i][new]]).reshape(-1, HKV, 128)
                    for i in range(2))
            used = at + 1
            assert -(-used // 16) * 16 == len(k)
            want, _, bound, _ = attention(rotated[b].cpu().numpy(), k[:used], v[:used],
                                          vc[b].cpu().numpy(), 128 ** -0.5)
            allowed = (np.abs(want) + bound[:, None]) * 2.0 ** -11 + bound[:, None] + 2.0 ** -24
            assert (np.abs(out[b].double().cpu().numpy() - want) <= allowed).all()
        ledger.commit_decode(batch)
    assert len(read_back) >= 4


def test_captured_steps_close_pages(cuda):
    """The steps of one page window to its last token: the replay that fills the page
    holds it in 4 bits, from rows that earlier replays stored."""
    from int4_helpers import held

    eager, graphed = (Served(cuda, [16, 160], 16) for _ in range(2))
    for _ in range(16):
        eager.prepare()
        eager.step()
        eager.advance()
    graphed.prepare()
    keep = [t.clone() for t in (graphed.tokens, *graphed.exact, graphed.codes, graphed.scales)]
    graphed.step()                                      # warm-up
    for t, was in zip((graphed.tokens, *graphed.exact, graphed.codes, graphed.scales), keep):
        t.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.step()
    pages = graphed.code_ids.long()
    for i in range(16):
        assert not graphed.prepare()
        before = graphed.codes[pages].clone()
        graph.replay()
        torch.cuda.synchronize()
        graphed.check()
        closed = ~(graphed.codes[pages] == before).flatten(1).all(1)
        assert closed.tolist() == [i == 15] * 2
        graphed.advance()
    assert graphed.length == [32, 176]
    for (codes, scales), ring in zip(unpack(graphed.codes, graphed.scales), graphed.exact):
        for b in range(2):
            want_codes, want_scales = held(ring[int(graphed.exact_ids[b])].float().cpu().numpy())
            np.testing.assert_array_equal(codes[int(pages[b])], want_codes)
            np.testing.assert_array_equal(scales[int(pages[b])], want_scales)
    for name in ("tokens", "history", "codes", "scales", "out", "lse", "shaped"):
        assert torch.equal(getattr(eager, name), getattr(graphed, name)), name
    assert all(torch.equal(a, b) for a, b in zip(eager.exact, graphed.exact))
