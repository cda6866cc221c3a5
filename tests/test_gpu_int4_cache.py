"""The writers and the reader-back of the cache held in 4 bits, bit for bit
against numpy, at lengths, strides and values where they could go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int4_helpers import held, unpack

pytestmark = pytest.mark.gpu


def _rows(tokens, heads, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, 128, generator=gen) * scale
    x[..., ::37] *= 8.0
    return x.half()


def _check_pages(codes, scales, page_ids, sources, centers, tokens):
    """Every written page against ``held`` of the centered float32 rows."""
    parts = unpack(codes, scales)
    for (got_codes, got_scales), source, center in zip(parts, sources, centers):
        x = source.float().numpy()
        if center is not None:
            x = x - center.float().numpy()
        want_codes, want_scales = held(x)
        for i, page in enumerate(page_ids):
            n = min(16, tokens - 16 * i)
            rows = slice(16 * i, 16 * i + n)
            np.testing.assert_array_equal(got_scales[page, :n], want_scales[rows])
            np.testing.assert_array_equal(got_codes[page, :n], want_codes[rows])
            assert not got_scales[page, n:].any()          # rows past the last token
            assert not got_codes[page, n:].any()


@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 33, 1000])
@pytest.mark.parametrize("heads", [1, 3, 8])
@pytest.mark.parametrize("centered", [True, False])
def test_quantize_pages(cuda, tokens, heads, centered):
    from pagegauge_amd import int4

    print(f"quantize tokens={tokens} heads={heads} centered={centered}", flush=True)
    k, v = _rows(tokens, heads, 1), _rows(tokens, heads, 2, 0.1)
    kc, vc = (_rows(1, heads, 3)[0], _rows(1, heads, 4)[0]) if centered else (None, None)
    pages = -(-tokens // 16)
    codes, scales = int4.allocate_pages(pages + 3, heads, cuda)
    ids = torch.randperm(pages + 3, generator=torch.Generator().manual_seed(5))[:pages].int()
    dev = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    untouched = [i for i in range(pages + 3) if i not in ids.tolist()]
    int4.quantize_pages(dev(k), dev(v), codes, scales, page_ids=ids.to(cuda), key_center=dev(kc),
                        value_center=dev(vc))
    _check_pages(codes, scales, ids.tolist(), (k, v), (kc, vc), tokens)
    assert not codes[untouched].any() and not scales[untouched].any()
    # back, whole and cut short, into rows of a wider projection
    parts = unpack(codes, scales)
    for count in {tokens, max(0, tokens - 5)}:
        wide = torch.full((count, 3 * heads * 128), 7.0, device=cuda, dtype=torch.float16)
        rows = [wide[:, j * heads * 128:(j + 1) * heads * 128].view(count, heads, 128) for j in (0, 2)]
        got = int4.dequantize_pages(codes, scales, ids.to(cuda), tokens=count, key_center=dev(kc),
                                    value_center=dev(vc), key=rows[0], value=rows[1])
        for out, (c, s), center in zip(got, parts, (kc, vc)):
            x = c[ids.tolist()].reshape(-1, heads, 128)[:count].astype(np.float32)
            x = x * s[ids.tolist()].reshape(-1, heads)[:count, :, None].astype(np.float32)
            if center is not None:
                x = x + center.float().numpy()
            assert torch.equal(out.cpu(), torch.from_numpy(x.astype(np.float16)))
        assert (wide[:, heads * 128:2 * heads * 128] == 7.0).all()


def test_quantize_strides_and_exact_pages(cuda):
    """Token rows of a fused projection, unaligned rows (the narrow loads), the
    identity table, skipped ids, and the FP16 copies of chosen pages."""
    from pagegauge_amd import int4

    heads, tokens = 2, 60
    k, v = _rows(tokens, heads, 1), _rows(tokens, heads, 2)
    kc, vc = _rows(1, heads, 3)[0], _rows(1, heads, 4)[0]
    fused = torch.cat((k.flatten(1), v.flatten(1)), dim=1).to(cuda)
    views = [fused[:, :256].view(tokens, heads, 128), fused[:, 256:].view(tokens, heads, 128)]
    odd = [torch.empty(t.numel() + 1, device=cuda, dtype=torch.float16)[1:].view(t.shape).copy_(t)
           for t in (k, v)]
    for sources in (views, odd):
        codes, scales = int4.allocate_pages(4, heads, cuda)
        ring = [torch.full((5, 16, heads, 128), 3.0, device=cuda, dtype=torch.float16) for _ in range(2)]
        exact_ids = torch.tensor([-1, 4, 9, 0], device=cuda, dtype=torch.int32)     # 9: outside
        int4.quantize_pages(*sources, codes, scales, key_center=kc.to(cuda), value_center=vc.to(cuda),
                            exact_page_ids=exact_ids, exact_key=ring[0], exact_value=ring[1])
        _check_pages(codes, scales, range(4), (k, v), (kc, vc), tokens)
        for pages, x, c in zip(ring, (k, v), (kc, vc)):
            want = torch.full((5, 16, heads, 128), 3.0).half()
            centered = (x.float() - c.float()).half()
            want[4] = centered[16:32]
            want[0, :12] = centered[48:60]
            assert torch.equal(pages.cpu(), want)
    codes, scales = int4.allocate_pages(4, heads, cuda)
    ids = torch.tensor([2, -1, 4, 0], device=cuda, dtype=torch.int32)      # -1 and 4: skipped
    int4.quantize_pages(*views, codes, scales, page_ids=ids)
    assert not codes[[1, 3]].any() and scales[0].any() and scales[2].any()
    back = int4.dequantize_pages(codes, scales, ids)[0]
    assert not back[16:48].any() and back[:16].any()
    int4.quantize_pages(views[0][:0], views[1][:0], codes, scales)         # no token


def test_quantize_extreme_values(cuda):
    """Zeros, subnormals, the largest values, infinities and NaN."""
    from pagegauge_amd import int4

    x = torch.zeros(16, 1, 128).half()
    x[1] = 2.0 ** -24
    x[2, 0, 5] = 65504.0
    x[2, 0, 6] = -65504.0 / 2
    x[3, 0, ::2], x[3, 0, 1::2] = 3.5, -3.5
    x[3, 0, 0] = 7.0                                       # halves of a step of 1
    x[4, 0, 1] = float("inf")
    x[4, 0, 2] = -1.0
    x[5, 0, 0], x[5, 0, 1] = float("nan"), 2.0
    x[6] = float("nan")
    codes, scales = int4.allocate_pages(1, 1, cuda)
    int4.quantize_pages(x.to(cuda), x.to(cuda), codes, scales)
    _check_pages(codes, scales, [0], (x, x), (None, None), 16)


@pytest.mark.parametrize("batch,q_heads,kv_heads", [(1, 4, 1), (7, 32, 8), (3, 6, 6), (2, 40, 5)])
@pytest.mark.parametrize("layout,part,scaling", [("half", 128, "none"), ("interleaved", 64, "linear")])
def test_rope_append(cuda, batch, q_heads, kv_heads, layout, part, scaling):
    from pagegauge_amd import int4, rotary
    from test_gpu_rotary import _check, _turned

    print(f"append batch={batch} heads={q_heads}/{kv_heads} {layout} {part}", flush=True)
    emb = rotary.RotaryEmbedding(128, part, layout=layout, scaling=scaling, factor=4.0)
    f = rotary.frequencies(part, 1.0e6, scaling, 4.0)
    gen = torch.Generator().manual_seed(batch)
    qkv = torch.randn(batch, (q_heads + 2 * kv_heads) * 128, generator=gen).half().to(cuda)
    q = qkv[:, :q_heads * 128].view(batch, q_heads, 128)
    k = qkv[:, q_heads * 128:(q_heads + kv_heads) * 128].view(batch, kv_heads, 128)
    v = qkv[:, (q_heads + kv_heads) * 128:].view(batch, kv_heads, 128)
    centers = [_rows(batch, kv_heads, s, 0.3).to(cuda) for s in (3, 4)]
    ring = [_rows((batch + 1) * 16, kv_heads, s).view(batch + 1, 16, kv_heads, 128).to(cuda) for s in (5, 6)]
    before = [t.clone() for t in ring]
    codes, scales = int4.allocate_pages(batch + 2, kv_heads, cuda)
    codes_before = codes.clone()
    positions = torch.tensor([(15, 4095, 0, 999999, 7, -1, 31)[i % 7] for i in range(batch)],
                             device=cuda, dtype=torch.int32)
    exact = torch.randperm(batch + 1, generator=gen)[:batch].int()
    code = torch.randperm(batch + 2, generator=gen)[:batch].int()
    rotated = torch.full((batch, q_heads, 128), 9.0, device=cuda, dtype=torch.float16)
    int4.rope_append(emb, q, k, v, positions, exact.to(cuda), code.to(cuda), *centers, rotated, *ring,
                     codes, scales)
    at = positions.tolist()
    live = [b for b in range(batch) if at[b] >= 0]
    _check(emb, f, q[live], positions[live], rotated[live])
    assert (rotated[[b for b in range(batch) if b not in live]] == 9.0).all()
    turned = _turned(emb, f, k.cpu(), positions.cpu())
    for pool, was, row, center, is_key in zip(ring, before, (turned, v.cpu().double()), centers, (1, 0)):
        want = was.cpu().double()
        for b in live:
            want[exact[b], at[b] % 16] = row[b] - center[b].cpu().double()
        # rounded once; the key's rotation as _check bounds it, each value's pair
        # sum at most twice the row's largest
        slack = 2.0 ** -20 * 2 * float(k.abs().max()) if is_key else 0.0
        off = (pool.cpu().double() - want).abs()
        assert (off <= want.abs() * 2.0 ** -11 * (1 + 2.0 ** -10) + 2.0 ** -25 + 1.001 * slack).all()
        touched = torch.zeros(batch + 1, 16, dtype=torch.bool)
        for b in live:
            touched[exact[b], at[b] % 16] = True
        assert torch.equal(pool.cpu()[~touched], was.cpu()[~touched])
    closing = [b for b in live if at[b] % 16 == 15]
    parts = unpack(codes, scales)
    for (got_codes, got_scales), pool in zip(parts, ring):
        for b in closing:
            want_codes, want_scales = held(pool[exact[b]].float().cpu().numpy())
            np.testing.assert_array_equal(got_codes[code[b]], want_codes)
            np.testing.assert_array_equal(got_scales[code[b]], want_scales)
    others = [p for p in range(batch + 2) if p not in [int(code[b]) for b in closing]]
    assert torch.equal(codes[others], codes_before[others]) and not scales[others].any()


@pytest.mark.parametrize("layout,part", [("half", 128), ("interleaved", 128), ("half", 66)])
def test_append_turns_as_rotate_does(cuda, layout, part):
    """The same bits of a query or key, whichever kernel turned it."""
    from pagegauge_amd import int4, rotary

    emb = rotary.RotaryEmbedding(128, part, layout=layout)
    batch, q_heads, kv_heads = 640, 8, 2
    q, k = _rows(batch, q_heads, 7).to(cuda), _rows(batch, kv_heads, 8).to(cuda)
    positions = (torch.arange(batch, dtype=torch.int32) * 7919 % 131072).to(cuda)
    want_q, want_k = emb.rotate(q, k, positions)
    ids = torch.arange(batch, dtype=torch.int32, device=cuda)
    none = torch.full_like(ids, -1)
    zeros = torch.zeros(batch, kv_heads, 128, dtype=torch.float16, device=cuda)
    rotated, (codes, scales) = torch.empty_like(q), int4.allocate_pages(1, kv_heads, cuda)
    ring = [torch.zeros(batch, 16, kv_heads, 128, dtype=torch.float16, device=cuda) for _ in range(2)]
    int4.rope_append(emb, q, k, k, positions, ids, none, zeros, zeros, rotated, *ring, codes, scales)
    assert torch.equal(rotated, want_q)
    assert torch.equal(ring[0][ids.long(), positions.long() % 16], want_k)


def test_append_skips_ids_outside_the_pools(cuda):
    from pagegauge_amd import int4, rotary

    emb = rotary.RotaryEmbedding(128)
    row = _rows(4, 1, 1).to(cuda)
    ring = [torch.zeros(2, 16, 1, 128, device=cuda, dtype=torch.float16) for _ in range(2)]
    codes, scales = int4.allocate_pages(2, 1, cuda)
    ids = lambda *a: torch.tensor(a, device=cuda, dtype=torch.int32)  # noqa: E731
    rotated = torch.zeros_like(row)
    int4.rope_append(emb, row, row, row, ids(15, 15, 15, 15), ids(-1, 2, 0, 1), ids(0, 1, -1, 2), row,
                     row, rotated, *ring, codes, scales)
    assert rotated.any(-1).all()
    assert ring[0][:, 15].any() and not ring[0][:, :15].any()
    assert not codes.any() and not scales.any()


def test_offsets_past_32_bits(cuda):
    """Pages of a pool of more than 4 GiB, and FP16 pages behind 4 GiB."""
    from pagegauge_amd import int4, rotary

    heads, pool = 8, 262144 + 8
    codes = torch.empty(pool, heads, 2, 1024, device=cuda, dtype=torch.uint8)
    scales = torch.empty(pool, heads, 4, 2, 4, device=cuda, dtype=torch.float16)
    k, v = _rows(48, heads, 1), _rows(48, heads, 2)
    ids = torch.tensor([pool - 1, 3, pool - 2], dtype=torch.int32)
    small = int4.allocate_pages(3, heads, cuda)
    int4.quantize_pages(k.to(cuda), v.to(cuda), codes, scales, page_ids=ids.to(cuda))
    int4.quantize_pages(k.to(cuda), v.to(cuda), *small)
    assert torch.equal(codes[ids.tolist()], small[0]) and torch.equal(scales[ids.tolist()], small[1])
    got = int4.dequantize_pages(codes, scales, ids.to(cuda))
    want = int4.dequantize_pages(*small)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ring = [torch.empty(131072 + 4, 16, heads, 128, device=cuda, dtype=torch.float16) for _ in range(2)]
    exact = torch.tensor([131072 + 3], device=cuda, dtype=torch.int32)
    for t, x in zip(ring, (k, v)):
        t[exact.long()] = x[:16].to(cuda)
    rotated = torch.empty(1, heads, 128, device=cuda, dtype=torch.float16)
    zero = torch.zeros(1, heads, 128, device=cuda, dtype=torch.float16)
    position = torch.tensor([31], device=cuda, dtype=torch.int32)
    last = [t[exact.long(), 15].clone() for t in ring]
    int4.rope_append(rotary.RotaryEmbedding(128), k[15:16].to(cuda), k[15:16].to(cuda),
                     v[15:16].to(cuda), position, exact, ids[:1].to(cuda), zero, zero, rotated, *ring,
                     codes, scales)
    assert torch.equal(ring[1][exact.long(), 15], last[1])
    assert torch.equal(ring[0][exact.long(), 15], rotated)
    parts = unpack(codes[pool - 1:], scales[pool - 1:])
    for (c, s), t in zip(parts, ring):
        want_c, want_s = held(t[exact.long()][0].float().cpu().numpy())
        np.testing.assert_array_equal(c[0], want_c)
        np.testing.assert_array_equal(s[0], want_s)
