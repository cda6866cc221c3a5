"""Rotary positions against the rotation in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _turned(emb, frequencies, x, positions):
    """The rotation of [T, H, D] rows in float64 (CPU)."""
    r = emb.rotary_dim
    angle = positions.double()[:, None] * frequencies
    cos, sin = (f(angle)[:, None, :] * emb.amplitude for f in (torch.cos, torch.sin))
    out = x.double().clone()
    where = ((slice(0, r // 2), slice(r // 2, r)) if emb.layout == "half"
             else (slice(0, r, 2), slice(1, r, 2)))
    a, b = (x.double()[..., w] for w in where)
    out[..., where[0]], out[..., where[1]] = a * cos - b * sin, b * cos + a * sin
    return out


def _check(emb, frequencies, x, positions, got):
    """Half a rounding of the row's type; the angle is reduced in 64 bits and
    rounded once (2^-25 of a turn, 2 pi 2^-25 < 2^-22), its sine and cosine are
    within 2^-22 and the products and sum round three times (2^-24 each): below
    2^-20 of the pair's absolute sum.  The angle itself, in radians, is off by
    2^-51 of its size: revolutions per position round twice (f / 2 pi), their
    product with the position once, and the angle here once, 2^-53 each.  2^-25
    is half a subnormal step of FP16."""
    x, positions, got = x.cpu(), positions.cpu(), got.cpu().double()
    want = _turned(emb, frequencies, x, positions)
    r = emb.rotary_dim
    size = x.double().abs()
    pair = torch.zeros_like(size)
    if emb.layout == "half":
        both = size[..., :r // 2] + size[..., r // 2:r]
        pair[..., :r // 2], pair[..., r // 2:r] = both, both
    else:
        both = size[..., 0:r:2] + size[..., 1:r:2]
        pair[..., 0:r:2], pair[..., 1:r:2] = both, both
    angle = torch.zeros_like(size)
    turned = (positions.double().abs()[:, None] * frequencies)[:, None, :].expand(*size.shape[:2], r // 2)
    if emb.layout == "half":
        angle[..., :r // 2], angle[..., r // 2:r] = turned, turned
    else:
        angle[..., 0:r:2], angle[..., 1:r:2] = turned, turned
    eps = torch.finfo(x.dtype).eps
    allowed = pair * abs(emb.amplitude) * angle * 2.0 ** -51 + want.abs() * eps / 2 * (1 + eps) + pair * abs(emb.amplitude) * 2.0 ** -20 + (
        2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    assert ((got - want).abs() <= allowed).all()
    assert torch.equal(got[..., r:], x[..., r:].double())


def _rows(device, dtype, tokens, heads, dim, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(tokens, heads, dim, generator=gen).to(dtype).to(device)


# vectors of 8, 4, 2 and 1 of the 16-bit types and 4, 2, 1 of float32; copied dims
@pytest.mark.parametrize("dim,part", [(128, 128), (128, 64), (96, 40), (64, 20), (80, 6), (256, 256),
                                      (2, 2), (10, 4)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rotation(cuda, dim, part, layout, dtype):
    from pagegauge_amd import rotary

    print(f"rotary dim={dim} part={part} {layout} {dtype}", flush=True)
    emb = rotary.RotaryEmbedding(dim, part, 1.0e4, layout)
    f = rotary.frequencies(part, 1.0e4)
    positions = torch.tensor([0, 1, 17, 4095, 1000003, 2 ** 31 - 1, 5], device=cuda,
                             dtype=torch.int32)
    q, k = _rows(cuda, dtype, 7, 6, dim, 1), _rows(cuda, dtype, 7, 2, dim, 2)
    oq, ok = emb.rotate(q, k, positions)
    _check(emb, f, q, positions, oq)
    _check(emb, f, k, positions, ok)
    # in place, the same bits
    q2, k2 = q.clone(), k.clone()
    assert emb.rotate(q2, k2, positions, q2, k2)[0] is q2
    assert torch.equal(q2, oq) and torch.equal(k2, ok)


# tokens and heads of one workgroup, of several, of a last one that is not full;
# sines of one token that fill the LDS; a vector of copied dims per head
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,part", [
    (1, 1, 0, 2, 2), (3, 70, 3, 128, 128), (130, 290, 10, 256, 256), (2, 3, 1, 16384, 16384),
    (2, 3, 1, 16384, 2), (5001, 13, 1, 64, 32), (2, 9000, 1, 4, 2), (70001, 1, 1, 16, 16)])
def test_rows_of_any_count(cuda, tokens, q_heads, kv_heads, dim, part):
    from pagegauge_amd import rotary

    print(f"rotary tokens={tokens} heads={q_heads}/{kv_heads} dim={dim} part={part}", flush=True)
    emb = rotary.RotaryEmbedding(dim, part, 1.0e4, "interleaved" if tokens % 2 else "half")
    f = rotary.frequencies(part, 1.0e4)
    positions = torch.arange(tokens, device=cuda, dtype=torch.int64) * 101
    q = _rows(cuda, torch.float16, tokens, q_heads, dim, 3)
    k = _rows(cuda, torch.float16, tokens, kv_heads, dim, 4) if kv_heads else None
    oq, ok = emb.rotate(q, k, positions)
    _check(emb, f, q, positions, oq)
    if kv_heads:
        _check(emb, f, k, positions, ok)


@pytest.mark.parametrize("scaling,factor", [("linear", 8.0), ("ntk", 4.0), ("by_parts", 16.0)])
def test_scalings(cuda, scaling, factor):
    from pagegauge_amd import rotary

    kwargs = dict(scaling=scaling, factor=factor, original_context=8192)
    emb = rotary.RotaryEmbedding(128, theta=1.0e6, **kwargs)
    assert emb.amplitude == (0.1 * math.log(factor) + 1.0 if scaling == "by_parts" else 1.0)
    positions = torch.arange(100000, 100033, device=cuda)          # int64
    q = _rows(cuda, torch.float32, 33, 4, 128, 3)
    got, none = emb.rotate(q, None, positions)
    assert none is None
    _check(emb, rotary.frequencies(128, 1.0e6, **kwargs), q, positions, got)


def test_strides_and_single_rows(cuda):
    """Slices of a fused projection, head-major rows, rows that are not 16-byte
    aligned, one token, many tokens and none."""
    from pagegauge_amd import rotary

    emb = rotary.RotaryEmbedding(128)
    f = rotary.frequencies(128, 1.0e6)
    gen = torch.Generator().manual_seed(5)
    for tokens in (1, 3, 1025):
        positions = torch.arange(tokens, device=cuda, dtype=torch.int32) * 31
        qkv = torch.randn(tokens, 12 * 128, generator=gen).half().to(cuda)
        q, k = qkv[:, :1024].view(tokens, 8, 128), qkv[:, 1024:1280].view(tokens, 2, 128)
        oq, ok = emb.rotate(q, k, positions)
        _check(emb, f, q, positions, oq)
        _check(emb, f, k, positions, ok)
        head_major = torch.empty(8, tokens, 128, device=cuda, dtype=torch.float16)
        emb.rotate(q, None, positions, head_major.transpose(0, 1))
        assert torch.equal(head_major.transpose(0, 1), oq)
        odd = torch.empty(tokens * 8 * 128 + 1, device=cuda, dtype=torch.float16)[1:].view(tokens, 8, 128)
        odd.copy_(q)
        assert torch.equal(emb.rotate(odd, None, positions)[0], oq)
    empty = torch.empty(0, 8, 128, device=cuda, dtype=torch.float16)
    assert emb.rotate(empty, None, positions[:0])[0].shape == (0, 8, 128)
    # an input broadcast over heads
    one = _rows(cuda, torch.float16, 3, 1, 128, 9)
    wide = emb.rotate(one.expand(3, 4, 128), None, positions[:3])[0]
    assert torch.equal(wide, emb.rotate(one, None, positions[:3])[0].expand(3, 4, 128))


def test_infinities_stay_in_their_pair(cuda):
    from pagegauge_amd import rotary

    emb = rotary.RotaryEmbedding(128, 64)
    x = _rows(cuda, torch.float16, 2, 1, 128, 4)
    x[0, 0, 3] = float("inf")
    x[1, 0, 100] = float("nan")                    # past the rotated part
    got = emb.rotate(x, None, torch.tensor([9, 9], device=cuda, dtype=torch.int32))[0].cpu()
    bad = ~torch.isfinite(got)
    assert bad[0, 0].nonzero().flatten().tolist() == [3, 35]
    assert bad[1, 0].nonzero().flatten().tolist() == [100]


def test_negative_positions_and_missing_heads(cuda):
    """Positions below zero turn back; a call without query heads turns the keys."""
    from pagegauge_amd import rotary

    emb = rotary.RotaryEmbedding(128, 96, layout="interleaved")
    f = rotary.frequencies(96, 1.0e6)
    x = _rows(cuda, torch.float32, 3, 2, 128, 6)
    positions = torch.tensor([-1, -70000, -2 ** 40], device=cuda)
    _check(emb, f, x, positions, emb.rotate(x, None, positions)[0])
    none, got = emb.rotate(x[:, :0], x, positions)
    assert none.shape == (3, 0, 128)
    assert torch.equal(got, emb.rotate(x, None, positions)[0])


def test_tensors_of_another_device_are_refused(cuda):
    from pagegauge_amd import rotary

    x = _rows(cuda, torch.float16, 1, 1, 128, 1)
    with pytest.raises(ValueError, match="current CUDA device"):
        rotary.RotaryEmbedding(128).rotate(x, None, torch.zeros(1, dtype=torch.int32))
