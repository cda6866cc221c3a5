"""Attention over the cache held in 4 bits against float64.

Tolerances.  A score is an exact product of FP16 queries with small integers
summed in float32 (128 additions, and 8 more roundings for scales), so its
error in base 2 is at most 136 * 2^-24 of sum |q||k| sm log2(e); a weight is off by ln 2
times that, and by 2^-20 for exp2 and the two-part FP16 probability.  An
output is a weighted mean, off by at most twice the weights' error times the
largest |v|, then rounded to FP16 (2^-11).  lse is off by the score's error and
a few float32 roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int4_helpers import attention, nibble_maps, random_pool, unpack

pytestmark = pytest.mark.gpu


class Case:
    """A batch over shuffled pools: ``history`` and ``tail`` tokens per request."""

    def __init__(self, cuda, history, tail, kv_heads, group, seed=1, with_tail=True, scale=0.3):
        from pagegauge_amd import int4

        gen = torch.Generator().manual_seed(seed)
        self.batch, self.hkv, self.group = len(history), kv_heads, group
        self.history, self.tail = history, tail
        tables = []
        for tokens in (history, tail):
            pages = [-(-t // 16) for t in tokens]
            indptr = torch.tensor([0] + list(np.cumsum(pages)), dtype=torch.int32)
            ids = torch.randperm(sum(pages) + 2, generator=gen)[:sum(pages)].int()
            last = torch.tensor([(t - 1) % 16 + 1 if t else 0 for t in tokens], dtype=torch.int32)
            tables.append((indptr, ids.to(cuda), last.to(cuda)))
        self.tables = tables
        self.codes, self.scales = random_pool(gen, len(tables[0][1]) + 2, kv_heads, cuda, scale)
        self.exact = [torch.randn(len(tables[1][1]) + 2, 16, kv_heads, 128, generator=gen).half().to(cuda)
                      for _ in range(2)]
        self.q = torch.randn(self.batch, kv_heads * group, 128, generator=gen).half().to(cuda)
        self.center = torch.randn(self.batch, kv_heads, 128, generator=gen).half().to(cuda)
        self.decode = int4.Int4PagedDecode(torch.empty(64 << 20, device=cuda, dtype=torch.uint8))
        self.with_tail = with_tail
        self.decode.plan(*tables[0], *(tables[1] if with_tail else ()),
                         num_qo_heads=kv_heads * group, num_kv_heads=kv_heads)

    def run(self, **over):
        a = dict(q=self.q, codes=self.codes, scales=self.scales,
                 exact_cache=self.exact if self.with_tail else None, value_center=self.center,
                 return_lse=True)
        a.update(over)
        return self.decode.run(**a)

    def check(self, out, lse, center=True, sm_scale=128 ** -0.5, q=None):
        out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        (kc, ks), (vc, vs) = unpack(self.codes, self.scales)
        pools = [(kc * ks.astype(np.float64)[..., None], vc * vs.astype(np.float64)[..., None]),
                 tuple(t.double().cpu().numpy() for t in self.exact)]
        for b in range(self.batch):
            k, v = [], []
            segments = (self.history, self.tail) if self.with_tail else (self.history,)
            for tokens, (indptr, ids, _), pool in zip(segments, self.tables, pools):
                pages = ids.cpu().numpy()[indptr[b]:indptr[b + 1]]
                k.append(pool[0][pages].reshape(-1, self.hkv, 128)[:tokens[b]])
                v.append(pool[1][pages].reshape(-1, self.hkv, 128)[:tokens[b]])
            want, want_lse, bound, lse_bound = attention(
                (self.q if q is None else q)[b].cpu().numpy(), np.concatenate(k), np.concatenate(v),
                self.center[b].cpu().numpy() if center else None, sm_scale)
            allowed = (np.abs(want) + bound[:, None]) * 2.0 ** -11 + bound[:, None] + 2.0 ** -24
            assert (np.abs(out[b] - want) <= allowed).all(), (b, np.abs(out[b] - want).max())
            if len(np.concatenate(k)):
                # the roundings alone: half a step of FP16 for each value
                assert np.linalg.norm(out[b] - want) <= 2.0 ** -11 * np.linalg.norm(want) * 1.01
                assert (np.abs(lse[b] - want_lse) <= lse_bound + 2.0 ** -20 + 2.0 ** -22 * np.abs(want_lse)).all()
            else:
                assert np.isneginf(lse[b]).all()


# up to 8 query heads per KV head, and more
both_forms = pytest.mark.parametrize("kv_heads,group", [(8, 4), (2, 16)])


# one token, inside a page, whole groups of pages, several items, past an item's pages
@pytest.mark.parametrize("history,tail", [
    ([1], [0]), ([0], [1]), ([17], [15]), ([64], [33]), ([512], [256]), ([4000], [256]),
    ([9001], [16]), ([0, 1, 300, 0, 65, 2048], [0, 0, 256, 40, 17, 250])])
@both_forms
def test_lengths(cuda, history, tail, kv_heads, group):
    print(f"attention history={history} tail={tail} heads={kv_heads}x{group}", flush=True)
    c = Case(cuda, history, tail, kv_heads, group)
    c.check(*c.run())


@pytest.mark.parametrize("kv_heads,group", [(8, 1), (5, 3), (1, 6), (4, 8), (2, 9), (2, 16), (16, 2)])
@pytest.mark.parametrize("with_tail", [True, False])
def test_head_layouts(cuda, kv_heads, group, with_tail):
    print(f"attention heads={kv_heads}x{group} tail={with_tail}", flush=True)
    c = Case(cuda, [700, 90], [100, 16], kv_heads, group, with_tail=with_tail)
    c.check(*c.run())


def test_large_batch_of_single_items(cuda):
    gen = torch.Generator().manual_seed(3)
    history = torch.randint(0, 500, (300,), generator=gen).tolist()
    tail = torch.randint(0, 60, (300,), generator=gen).tolist()
    c = Case(cuda, history, tail, 2, 4)
    c.check(*c.run())


def test_no_center_given_outputs_and_strides(cuda):
    c = Case(cuda, [300, 40], [20, 0], 8, 4)
    out, lse = c.run(value_center=None)
    c.check(out, lse, center=False)
    wide = torch.empty(2, 48, 128, device=cuda, dtype=torch.float16)
    wide[:, :32] = c.q
    given = torch.empty_like(out)
    given_lse = torch.empty_like(lse)
    got = c.run(q=wide[:, :32], value_center=None, out=given, lse=given_lse, return_lse=False)
    assert got is given and torch.equal(given, out) and torch.equal(given_lse, lse)
    scaled, slse = c.run(sm_scale=0.5)
    c.check(scaled, slse, sm_scale=0.5)


@pytest.mark.parametrize("scale", [2.0 ** -14, 2000.0])
@both_forms
def test_scales_of_any_size(cuda, scale, kv_heads, group):
    """Values far below and above 1 beside exact ones near 1."""
    c = Case(cuda, [500, 20], [30, 0], kv_heads, group, scale=scale)
    c.scales[..., 0, :] = 0.1           # K's
    c.check(*c.run())


@both_forms
def test_scores_far_apart(cuda, kv_heads, group):
    """One token outweighs all others by any factor; all tokens alike."""
    c = Case(cuda, [900], [60], kv_heads, group)
    c.q *= 30.0
    c.check(*c.run())
    c.q.zero_()
    c.check(*c.run())


@both_forms
def test_what_lies_behind_the_last_token_is_not_read(cuda, kv_heads, group):
    """NaN and infinities in the masked rows of both kinds of pages."""
    c = Case(cuda, [37, 530], [21, 5], kv_heads, group)
    want = c.run()
    for b in range(2):
        page = int(c.tables[0][1][int(c.tables[0][0][b + 1]) - 1])
        used = (c.history[b] - 1) % 16 + 1
        rows = c.scales[page].view(kv_heads, 4, 2, 4)
        for t in range(used, 16):
            rows[:, t // 4, :, t % 4] = float("nan") if t % 2 else float("inf")
        page = int(c.tables[1][1][int(c.tables[1][0][b + 1]) - 1])
        used = (c.tail[b] - 1) % 16 + 1
        c.exact[0][page, used:] = float("nan")
        c.exact[1][page, used:] = float("inf")
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_lengths_are_read_on_the_device(cuda):
    """The last lengths move between runs of one plan, down to no token."""
    c = Case(cuda, [48, 700], [16, 30], 8, 4)
    c.check(*c.run())
    c.tables[0][2].copy_(torch.tensor([5, 1]))
    c.tables[1][2].copy_(torch.tensor([3, 16]))
    c.history, c.tail = [37, 689], [3, 32]
    c.check(*c.run())
    lone = Case(cuda, [7], [0], 8, 4)
    lone.tables[0][2].zero_()
    out, lse = lone.run()
    assert torch.equal(out, lone.center.repeat_interleave(4, dim=1)) and torch.isneginf(lse).all()


@pytest.mark.parametrize("group", [4, 16])
def test_infinite_scores(cuda, group):
    """Scores of -inf leave the others; a NaN score makes its head NaN."""
    c = Case(cuda, [0], [40], 1, group)
    c.q[:] = 1.0
    c.exact[0].fill_(0.25)
    first = int(c.tables[1][1][0])
    c.exact[0][first, :, 0, 0] = float("-inf")        # the whole first page
    out, lse = c.run()
    v = c.exact[1][c.tables[1][1].long()].reshape(-1, 128)[16:40].double()
    want = v.mean(0) + c.center[0, 0].double()
    assert ((out[0].double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -18).all()
    c.exact[0][first, :, 0, 0] = 0.25
    c.q[0, 2, 0] = float("nan")
    out, lse = c.run()
    assert out[0, 2].isnan().all() and out[0, [h for h in range(group) if h != 2]].isfinite().all()


def test_pool_past_4_gib(cuda):
    """Pages at byte offsets past 32 bits."""
    from pagegauge_amd import int4

    c = Case(cuda, [200], [20], 8, 4)
    pool = 262144 + 16
    codes = torch.empty(pool, 8, 2, 1024, device=cuda, dtype=torch.uint8)
    scales = torch.empty(pool, 8, 4, 2, 4, device=cuda, dtype=torch.float16)
    pages = c.codes.shape[0]
    codes[pool - pages:], scales[pool - pages:] = c.codes, c.scales
    want = c.run()
    c.tables[0][1].add_(pool - pages)
    got = c.run(codes=codes, scales=scales)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert isinstance(c.decode, int4.Int4PagedDecode)


def test_graphs_sharing_a_workspace_and_streams(cuda):
    """Two captured runs of one object replayed in turn beside eager work, and
    a run on another stream."""
    c = Case(cuda, [3000, 100], [200, 16], 8, 4)
    q2 = c.q.flip(0).contiguous()
    want = [c.run(), c.run(q=q2)]
    outs = [(torch.empty_like(want[0][0]), torch.empty_like(want[0][1])) for _ in range(2)]
    graphs = []
    for q, (out, lse) in zip((c.q, q2), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.run(q=q, out=out, lse=lse)
        graphs.append(graph)
    for _ in range(3):
        for graph, (out, lse), (want_out, want_lse) in zip(graphs, outs, want):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want_out) and torch.equal(lse, want_lse)
        assert torch.equal(c.run()[0], want[0][0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = c.run()
    stream.synchronize()
    assert torch.equal(got[0], want[0][0])


def _set_nibbles(c, part, codes):
    """Puts ``codes`` [tokens, Hkv, 128] into the history's pages as K (0) or V (1)."""
    where = nibble_maps()[part]
    ids = c.tables[0][1].cpu().numpy()
    nibbles = np.full((c.codes.shape[0], c.hkv, 2048), 8, np.uint8)
    rows = codes.reshape(len(ids), 16, c.hkv, 128).transpose(0, 2, 1, 3)
    nibbles[ids] = (rows[:, :, where[:, 0], where[:, 1]] + 8).astype(np.uint8)
    c.codes[:, :, part] = torch.from_numpy(nibbles[..., ::2] | nibbles[..., 1::2] << 4).to(c.codes.device)


@both_forms
def test_a_value_among_zeros_keeps_its_bits(cuda, kv_heads, group):
    """Values of code 0 add nothing, however many: 4096 tokens of one item weigh alike,
    and each channel has one value that is not 0, of code 1 or -1 and its token's
    scale.  The output is scale / 4096 but for the rounding of the probabilities' sum,
    a chain of fewer than 700 additions of 2^-24 each (below 2^-14), of a probability,
    its product with the scale, the join of 4 waves and the quotient (below 2^-18
    together), and FP16's 2^-11."""
    tokens = 4096
    c = Case(cuda, [tokens], [0], kv_heads, group, with_tail=False)
    c.decode.plan(*c.tables[0], num_qo_heads=kv_heads * group, num_kv_heads=kv_heads, num_cus=1)
    assert c.decode.num_work_items == 1
    c.q.zero_()
    gen = torch.Generator().manual_seed(8)
    # scales of 11 bits from 1 to 128: exact products, outputs that are no subnormals
    c.scales.copy_(torch.randint(1024, 2048, c.scales.shape, generator=gen)
                   * 2.0 ** -torch.randint(4, 11, c.scales.shape, generator=gen))
    at = torch.randint(0, tokens, (kv_heads, 128), generator=gen).numpy()
    sign = (torch.randint(0, 2, (kv_heads, 128), generator=gen) * 2 - 1).numpy()
    codes = np.zeros((tokens, kv_heads, 128), np.int64)
    for h in range(kv_heads):
        codes[at[h], h, np.arange(128)] = sign[h]
    _set_nibbles(c, 1, codes)
    out, _ = c.run(value_center=None)
    scales = unpack(c.codes, c.scales)[1][1].astype(np.float64)                # [pages, 16, Hkv]
    pages = c.tables[0][1].cpu().numpy()
    want = np.repeat([sign[h] * scales[pages[at[h] // 16], at[h] % 16, h] / tokens
                      for h in range(kv_heads)], group, axis=0)
    got = out[0].double().cpu().numpy()
    assert (np.abs(got - want) <= np.abs(want) * (2.0 ** -11 + 2.0 ** -14 + 2.0 ** -17)).all()


@both_forms
def test_small_products_beside_large_ones(cuda, kv_heads, group):
    """Requests of one token whose key has two codes of 1 or -1 that meet query values of
    1 to 2 and of 2^-10 to 2^-9: the dot has 22 bits, so no order of float32 sums
    rounds it.  lse is that dot times the scale, the softmax scale and log2(e): each
    product rounds once, their base twice more and its weight's exponent once, 2^-24
    of the score each and below 2^-21 together, and log2 of a weight near 1 is good to
    2^-20."""
    batch = 40
    c = Case(cuda, [1] * batch, [0] * batch, kv_heads, group, with_tail=False)
    gen = torch.Generator().manual_seed(9)
    q = torch.randn(batch, kv_heads * group, 128, generator=gen)
    codes = np.zeros((batch * 16, kv_heads, 128), np.int64)
    for b in range(batch):
        for h in range(kv_heads):
            large, small = torch.randperm(128, generator=gen)[:2].tolist()
            codes[16 * b, h, [large, small]] = (torch.randint(0, 2, (2,), generator=gen) * 2 - 1).numpy()
            rows = slice(h * group, (h + 1) * group)
            q[b, rows, large] = 1.0 + torch.rand(group, generator=gen)
            q[b, rows, small] = 2.0 ** -10 * (1.0 + torch.rand(group, generator=gen))
    c.q.copy_(q)
    _set_nibbles(c, 0, codes)
    out, lse = c.run(sm_scale=4.0)
    ids = c.tables[0][1].cpu().numpy()
    scales = unpack(c.codes, c.scales)[0][1].astype(np.float64)[ids, 0]            # [B, Hkv]
    dots = np.einsum("bhgd,bhd->bhg", c.q.double().cpu().numpy().reshape(batch, kv_heads, group, 128),
                     codes[::16].astype(np.float64))
    want = (dots * scales[..., None] * 4.0 * np.log2(np.e)).reshape(batch, -1)
    assert (np.abs(lse.double().cpu().numpy() - want) <= np.abs(want) * 2.0 ** -21 + 2.0 ** -20).all()


def test_gradients_are_refused(cuda):
    """The result would have no history: it is not computed, but for no_grad()."""
    c = Case(cuda, [40], [20], 2, 4)
    want = c.run()
    wanted = dict(q=c.q, value_center=c.center, exact_cache=c.exact)
    for name, t in wanted.items():
        t = ([x.clone().requires_grad_() for x in t] if name == "exact_cache"
             else t.clone().requires_grad_())
        with pytest.raises(ValueError, match="no gradient"):
            c.run(**{name: t})
        with torch.no_grad():
            assert torch.equal(c.run(**{name: t})[0], want[0])


@pytest.mark.parametrize("kv_heads,group", [(2, 4), (1, 16)])
@pytest.mark.parametrize("sm_scale", [128 ** -0.5, 2.0 ** 30, 2.0 ** 79])
@pytest.mark.parametrize("with_tail", [True, False])
def test_scores_of_any_size(cuda, kv_heads, group, sm_scale, with_tail):
    """Queries of +-2^15 and scales of 2^15: a score is 2^30 times a whole number, exact, so a
    weight is 1 or 0.  With a tail, whose keys are +-2^15 in all dims, it has the largest ones."""
    c = Case(cuda, [1000, 3000, 40, 0], [40, 0, 16, 300], kv_heads, group, with_tail=with_tail)
    c.q = torch.where(c.q[:, :, :1] > 0, 2.0 ** 15, -2.0 ** 15).half().expand(c.q.shape).contiguous()
    c.scales[:, :, :, 0] = 2.0 ** 15
    c.exact[0] = torch.where(c.exact[0][..., :1] > 0, 2.0 ** 15, -2.0 ** 15).half().expand(c.exact[0].shape).contiguous()
    out, lse = c.run(sm_scale=sm_scale)
    (kc, ks), (vc, vs) = unpack(c.codes, c.scales)
    pools = [(kc * ks.astype(np.float64)[..., None], vc * vs.astype(np.float64)[..., None]),
             tuple(t.double().cpu().numpy() for t in c.exact)]
    for b in range(c.batch):
        rows = [[p[ids.cpu().numpy()[indptr[b]:indptr[b + 1]]].reshape(-1, kv_heads, 128)[:tokens[b]] for p in pool]
                for tokens, (indptr, ids, _), pool in zip((c.history, c.tail)[:1 + with_tail], c.tables, pools)]
        k, v = (np.concatenate(x) for x in zip(*rows))
        for head in range(kv_heads * group):
            h = head // group
            center = c.center[b, h].double().cpu().numpy()
            got = out[b, head].double().cpu().numpy()
            if not len(k):
                assert np.array_equal(got, center) and float(lse[b, head]) == -np.inf
                continue
            s = k[:, h] @ c.q[b, head].double().cpu().numpy()
            top = s == s.max()
            want = v[top, h].mean(0) + center
            # equal weights in two parts (2^-20), sums of float32, the output's half step
            bound = (2.0 ** -19 + len(k) * 2.0 ** -24) * np.abs(v[:, h]).max()
            assert (np.abs(got - want) <= bound + np.abs(want) * 2.0 ** -11 + 2.0 ** -24).all(), (b, head)
            want_lse = s.max() * np.float64(np.float32(sm_scale)) * np.log2(np.e) + np.log2(top.sum())
            assert abs(float(lse[b, head]) - want_lse) <= 2.0 ** -21 * abs(want_lse), (b, head)
