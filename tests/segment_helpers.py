"""Batches over shared, own, selected and exact pages, and attention over them in 64
bits: what the kernels are held against.

Tolerances.  A score is an exact product of FP16 queries with FP16 values or whole
numbers, summed in float32 (128 additions, 8 more roundings for scales): its error in
base 2 is at most 136 * 2^-24 of sum |q||k| sm log2(e), and a weight is off by ln 2 times
that.  exp2, the two-part FP16 probability and its product with V's scale add 2^-20; a
kernel that takes the probability as one FP16 value adds half a step of it, 2^-11, or
where it is subnormal 2^-32 of the largest.  Sums of T tokens take at most T / 16 + 64
float32 additions, each off by 2^-24 of the sum.  An output is a weighted mean, off by at
most the weights' error times the largest |v| (twice where the sum of weights is off as
well), then rounded to FP16 (2^-11).  lse is off by the score's error and a few float32
roundings."""

from __future__ import annotations

import numpy as np
import torch

LOG2E = np.log2(np.e)


def table(lengths, gen, spare=2):
    """(host indptr, shuffled page ids, last lengths) of token counts."""
    pages = [-(-n // 16) for n in lengths]
    indptr = torch.tensor([0] + list(np.cumsum(pages)), dtype=torch.int32)
    ids = torch.randperm(sum(pages) + spare, generator=gen)[:sum(pages)].int()
    last = torch.tensor([(n - 1) % 16 + 1 if n else 0 for n in lengths], dtype=torch.int32)
    return indptr, ids, last


def int8_pool(gen, pages, heads, scale=0.02):
    """Codes over the whole of int8 and scales of [scale / 4, scale]."""
    codes = [torch.randint(-128, 128, (pages, 16, heads, 128), generator=gen).to(torch.int8) for _ in range(2)]
    scales = [((torch.rand(pages, heads, generator=gen) * 0.75 + 0.25) * scale).half() for _ in range(2)]
    return codes, scales


def values(cache, scale):
    """float64 [pages, 16, H, 128] of a pool."""
    x = cache.double().cpu().numpy()
    return x if scale is None else x * scale.double().cpu().numpy()[:, None, :, None]


def rows_of(pools, ids, tokens):
    """K and V [tokens, H, 128] of pages in order."""
    return [p[ids].reshape(-1, *p.shape[2:])[:tokens] for p in pools]


def check_head(out, lse, q, k, v, center, sm_scale, single_part):
    """One KV head of a request: out [G, 128] and lse [G] for q [G, 128], float64 k and v
    [T, 128]."""
    q = q.astype(np.float64)
    if len(k) == 0:
        want, bound, want_lse = np.zeros_like(q), 0.0, np.full(len(q), -np.inf)
    else:
        s = q @ k.T * (sm_scale * LOG2E)
        m = s.max(1, keepdims=True)
        p = np.exp2(s - m)
        total = p.sum(1, keepdims=True)
        want, want_lse = p @ v / total, (m + np.log2(total))[:, 0]
        spread = (np.abs(q) @ np.abs(k).T).max(1) * sm_scale * LOG2E
        score = 136 * 2.0 ** -24 * spread
        weight = 2 * (np.log(2.0) * score + 2.0 ** -20 + (len(k) / 16 + 64) * 2.0 ** -24)
        if single_part:
            weight += 2.0 ** -11 + len(k) * 2.0 ** -32
        bound = (weight * np.abs(v).max())[:, None]
        assert (np.abs(lse - want_lse) <= score + 2.0 ** -20 + 2.0 ** -22 * np.abs(want_lse)
                + (len(k) / 16 + 64) * 2.0 ** -24).all(), np.abs(lse - want_lse).max()
    if center is not None:
        want = want + center.astype(np.float64)
    allowed = (np.abs(want) + bound) * 2.0 ** -11 + bound + 2.0 ** -24
    assert (np.abs(out - want) <= allowed).all(), np.abs(out - want).max()
    if len(k) == 0:
        assert np.isneginf(lse).all()


class Batch:
    """Requests over shuffled pools.  ``segments``: (first, end, tokens) of prefixes;
    ``own`` and ``tail``: tokens per request."""

    def __init__(self, cuda, segments, own, tail, kv_heads, group, kind=torch.int8, seed=1, scale=0.02):
        gen = torch.Generator().manual_seed(seed)
        self.segments, self.own, self.tail = segments, own, tail
        self.batch, self.hkv, self.group, self.kind = len(own), kv_heads, group, kind
        self.prefix_ptr, _, prefix_last = table([s[2] for s in segments], gen)
        self.own_ptr, _, last = table(own, gen)
        shared = int(self.prefix_ptr[-1])
        pool = shared + int(self.own_ptr[-1]) + 3
        order = torch.randperm(pool, generator=gen).int()
        self.prefix_ids, self.ids = order[:shared].to(cuda), order[shared:pool - 3].to(cuda)
        self.prefix_last, self.last = prefix_last.to(cuda), last.to(cuda)
        self.tail_ptr, tail_ids, tail_last = table(tail, gen)
        self.tail_ids, self.tail_last = tail_ids.to(cuda), tail_last.to(cuda)
        if kind is torch.int8:
            cache, scales = int8_pool(gen, pool, kv_heads, scale)
            self.scales = [s.to(cuda) for s in scales]
        else:
            cache = [torch.randn(pool, 16, kv_heads, 128, generator=gen).half() for _ in range(2)]
            self.scales = [None, None]
        self.cache = [c.to(cuda) for c in cache]
        self.exact = [torch.randn(len(tail_ids) + 2, 16, kv_heads, 128, generator=gen).half().to(cuda)
                      for _ in range(2)]
        self.q = torch.randn(self.batch, kv_heads * group, 128, generator=gen).half().to(cuda)
        self.center = torch.randn(self.batch, kv_heads, 128, generator=gen).half().to(cuda)

    def own_table(self):
        return self.own_ptr, self.ids, self.last

    def tail_table(self):
        return self.tail_ptr, self.tail_ids, self.tail_last

    def keys_and_values(self, selected=None):
        """``f(b, h)``: float64 K and V [T, 128] that KV head h of request b sees."""
        pools = [values(c, s) for c, s in zip(self.cache, self.scales)]
        exact = [values(c, None) for c in self.exact]
        prefix_ids, ids, tail_ids = (t.cpu().numpy() for t in (self.prefix_ids, self.ids, self.tail_ids))
        prefix_last, last, tail_last = (t.tolist() for t in (self.prefix_last, self.last, self.tail_last))

        def part(pool, ptr, at, lasts, i, h, pages=None):
            begin, end = int(ptr[i]), int(ptr[i + 1])
            rows = []
            for page in range(end - begin) if pages is None else pages:
                if not 0 <= page < end - begin:
                    continue
                count = lasts[i] if page == end - begin - 1 else 16
                rows.append([p[at[begin + page], :count, h] for p in pool])
            return rows

        def seen(b, h):
            rows = []
            for i, (first, end, _) in enumerate(self.segments):
                if first <= b < end:
                    rows += part(pools, self.prefix_ptr, prefix_ids, prefix_last, i, h)
            pages = None if selected is None else selected[b, h]
            rows += part(pools, self.own_ptr, ids, last, b, h, pages)
            rows += part(exact, self.tail_ptr, tail_ids, tail_last, b, h)
            return [np.concatenate([r[i] for r in rows] + [np.zeros((0, 128))]) for i in range(2)]

        return seen

    def check(self, out, lse, center=True, sm_scale=128 ** -0.5, selected=None, q=None, requests=None,
              single_part=True):
        out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        q = (self.q if q is None else q).cpu().numpy()
        centers = self.center.cpu().numpy()
        seen = self.keys_and_values(selected)
        for b in range(self.batch) if requests is None else requests:
            for h in range(self.hkv):
                rows = slice(h * self.group, (h + 1) * self.group)
                check_head(out[b, rows], lse[b, rows], q[b, rows], *seen(b, h), centers[b, h] if center else None,
                           sm_scale, single_part)
