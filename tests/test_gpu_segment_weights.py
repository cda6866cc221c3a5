"""How many bits the weights of shared prefixes, own, selected and exact pages have.

Every query row is the same; queries are multiples of 2^-2 and keys of 2^-7, so that a score
before the softmax scale is exact.  Its weight is off by the scale's two roundings (2^-23 of the
distance to the largest score in base 2, at most ``spread``), that of its exponent (2^-24 of a
number below 64), exp2 and a product with V's scale (2^-22 together), and by its parts: 2^-23
of itself with two, with one 2^-11, or 2^-32 of the largest where that is subnormal.  T tokens are
summed with at most T / 16 + 64 additions in float32, each off by 2^-24 of the sum.  Weights and
sums are so off relative to sum p |v|, which the output is not: where values cancel it is
thousands of times smaller, and the two forms are told apart.  The sum of weights has the same
errors and is relative to the output; that is rounded to FP16 in the end (2^-11, or 2^-25)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import test_gpu_sparse as selecting
from segment_helpers import LOG2E, Batch
from test_gpu_prefix import planned, run

both_kinds = pytest.mark.parametrize("kind", [torch.int8, torch.float16])
SM = 128 ** -0.5


def allowed(p, v, two_parts):
    """Output [128] of weights p [T] and values v [T, 128] in 64 bits, and what it may be off by."""
    spread = np.log2(p.max() / p.min())
    weight = np.log(2.0) * (spread * 2.0 ** -23 + 2.0 ** -18) + 2.0 ** -22
    weight += 2.0 ** -23 if two_parts else 2.0 ** -11 + len(p) * 2.0 ** -32 * p.max() / p.sum()
    weight += (len(p) / 16 + 64) * 2.0 ** -24
    want = p @ v / p.sum()
    bound = weight * (p @ np.abs(v) / p.sum() + np.abs(want))
    return want, bound + np.maximum((np.abs(want) + bound) * 2.0 ** -11, 2.0 ** -25)


def quarters(gen, *shape):
    return torch.randint(-6, 7, shape, generator=gen).half() / 4


def weights_of(q, codes):
    """float64 [T] of one query row [128] over keys of codes [T, 128] times 2^-7."""
    s = codes @ q * (np.float64(np.float32(SM)) * LOG2E * 2.0 ** -7)
    return np.exp2(s - s.max())


def cancelling(p, scale, rng):
    """Whole numbers [T, 128] of at most 100 with sum p scale c near 0: the tokens that weigh most
    take the sign that the sum asks for, the last ones what is left of it."""
    c, total = np.zeros((len(p), 128)), np.zeros(128)
    order = np.argsort(-p * scale)
    for i, t in enumerate(order):
        w = p[t] * scale[t]
        sign = np.where(total > 0, -1.0, 1.0)
        c[t] = sign * rng.integers(20, 101, 128) if i < len(order) - 5 else np.clip(np.rint(-total / w), -100, 100)
        total += w * c[t]
    return c


class Exact:
    """Tokens in one place (prefix, own or exact pages), one query for all rows."""

    def __init__(self, cuda, place, requests, group, tokens, kind, values, kv_heads=2):
        at_place = lambda name: [tokens if place == name else 0] * requests  # noqa: E731
        b = Batch(cuda, [(0, requests, tokens)] if place == "prefix" else [], at_place("own"), at_place("tail"),
                  kv_heads, group, kind, seed=tokens)
        gen = torch.Generator().manual_seed(requests + group)
        rng = np.random.default_rng(7)
        q = quarters(gen, kv_heads, 128)
        b.q = q.repeat_interleave(group, 0).expand(requests, kv_heads * group, 128).contiguous().to(cuda)
        pools, ptr, ids = {"prefix": (b.cache, b.prefix_ptr, b.prefix_ids), "own": (b.cache, b.own_ptr, b.ids),
                           "tail": (b.exact, b.tail_ptr, b.tail_ids)}[place]
        codes = place != "tail" and kind is torch.int8
        if codes:
            b.scales[0].fill_(2.0 ** -7)
        self.b, self.weights, self.values = b, {}, {}
        for first in range(1 if place == "prefix" else requests):
            pages = ids[int(ptr[first]):int(ptr[first + 1])].cpu().long()
            page, slot = pages.repeat_interleave(16)[:tokens], torch.arange(16).repeat(len(pages))[:tokens]
            for h in range(kv_heads):
                k = torch.randint(-127, 128, (tokens, 128), generator=gen)
                p = weights_of(q[h].double().numpy(), k.double().numpy())
                scale = 2.0 ** -(6 + page % 2).double().numpy() if codes else np.full(tokens, 2.0 ** -6)
                c = values(p, scale, rng)
                pools[0][page, slot, h] = k.to(torch.int8).to(cuda) if codes else (k.half() / 128).to(cuda)
                v = torch.from_numpy(c)
                pools[1][page, slot, h] = v.to(torch.int8).to(cuda) if codes else (v / 64).half().to(cuda)
                if codes:
                    b.scales[1][page, h] = torch.from_numpy(scale).half().to(cuda)
                for r in range(requests) if place == "prefix" else (first,):
                    self.weights[r, h], self.values[r, h] = p, c * scale[:, None]

    def check(self, out, two_parts):
        b = self.b
        out = out.double().cpu().numpy().reshape(b.batch, b.hkv, b.group, 128)
        for r in range(b.batch):
            for h in range(b.hkv):
                want, bound = allowed(self.weights[r, h], self.values[r, h], two_parts)
                assert (np.abs(out[r, h] - want) <= bound).all(), (r, h, (np.abs(out[r, h] - want) / bound).max())


def one_value_a_channel(p, scale, rng):
    """Each channel has one value that is not 0: a token lost, or taken twice, is seen."""
    c = np.zeros((len(p), 128))
    edges = np.array([t for t in (0, 15, 16, 63, 64, len(p) - 1) if t < len(p)])
    c[np.concatenate((edges, rng.integers(0, len(p), 128)))[:128], np.arange(128)] = 100
    return c


VALUES = {"cancelling": (cancelling, 40), "one a channel": (one_value_a_channel, 5003)}
both_values = pytest.mark.parametrize("values,tokens", VALUES.values(), ids=VALUES)


@pytest.mark.parametrize("kind", [torch.int8, torch.float16])
def test_one_part_is_told_from_two(kind):
    """The bound of two parts, on the CPU: a model with one FP16 value per weight passes it, many
    times over, and one with the remainder in a second stays within."""
    rng = np.random.default_rng(3)
    gen = torch.Generator().manual_seed(3)
    q, k = quarters(gen, 128).double().numpy(), torch.randint(-127, 128, (40, 128), generator=gen).double().numpy()
    p = weights_of(q, k)
    scale = 2.0 ** -(6.0 + np.arange(40) // 16 % 2) if kind is torch.int8 else np.full(40, 2.0 ** -6)
    c = cancelling(p, scale, rng)
    w = (p * scale if kind is torch.int8 else p) * 2.0 ** 10
    rest = scale if kind is torch.float16 else np.ones(40)
    want, bound = allowed(p, c * scale[:, None], True)
    one = w.astype(np.float16).astype(np.float64)
    two = one + (w - one).astype(np.float16).astype(np.float64)
    off = [np.abs((x * rest) @ c / (p.sum() * 2.0 ** 10) - want) / bound for x in (one, two)]
    assert off[0].max() > 8 and off[1].max() < 1, [x.max() for x in off]
    assert (np.abs((one * rest) @ c / (p.sum() * 2.0 ** 10) - want) <= allowed(p, c * scale[:, None], False)[1]).all()


# 4, 16 and 32 query rows per KV head without tiles, 36 over tiles of two waves' rows, 80 of four
@pytest.mark.gpu
@pytest.mark.parametrize("requests", [1, 4, 8, 9, 20])
@both_values
@both_kinds
def test_prefixes(cuda, requests, values, tokens, kind):
    from pagegauge_amd import prefix

    print(f"weights prefix {requests} {tokens} {kind}", flush=True)
    e = Exact(cuda, "prefix", requests, 4, tokens, kind, values)
    _, items, _, _ = prefix.plan_work_items(e.b.own_ptr, None, [(0, requests)], e.b.prefix_ptr, 8, 2, kind)
    tiles = items[:, 14] > 16
    assert bool(tiles.any()) == (requests > 8)
    e.check(run(planned(e.b, cuda, with_tail=False), e.b, exact_cache=None, value_center=None, return_lse=False),
            two_parts=not bool(tiles.any()))


@pytest.mark.gpu
@pytest.mark.parametrize("group", [4, 16])
@pytest.mark.parametrize("place", ["own", "tail"])
@both_values
@both_kinds
def test_own_and_exact_pages(cuda, group, place, values, tokens, kind):
    print(f"weights {place} {group} {tokens} {kind}", flush=True)
    e = Exact(cuda, place, 3, group, tokens, kind, values)
    e.check(run(planned(e.b, cuda), e.b, value_center=None, return_lse=False), two_parts=True)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [4, 16])
@both_values
def test_selected_pages(cuda, group, values, tokens):
    """All pages selected, and they go through the selection."""
    print(f"weights selected {group} {tokens}", flush=True)
    e = Exact(cuda, "own", 3, group, tokens, torch.int8, values)
    decode = selecting.planned(e.b, cuda, -(-tokens // 16))
    selected = decode.select(e.b.q, selecting.bounds_of(e.b, cuda), e.b.scales[0])
    out = selecting.run(decode, e.b, selected, value_center=None, return_lse=False)
    e.check(out, two_parts=True)
