"""Rotary frequencies against closed forms, and what the operator refuses."""

from __future__ import annotations

import math

import pytest
import torch

from pagegauge_amd import _capi, rotary


def test_frequencies():
    f = rotary.frequencies(8, 10000.0)
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(rotary.frequencies(8, 1e4, "linear", 4.0), f / 4, rtol=1e-15)
    # the base raised keeps the fastest pair and stretches the slowest by the factor
    ntk = rotary.frequencies(8, 1e4, "ntk", 4.0)
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), 0.001 / 4, rel_tol=1e-12)


def test_by_parts_keeps_fast_pairs_and_stretches_slow_ones():
    r, theta, context, factor = 128, 1.0e4, 4096, 8.0
    f = rotary.frequencies(r, theta)
    got = rotary.frequencies(r, theta, "by_parts", factor, context)
    turns = f * context / (2 * math.pi)
    assert torch.equal(got[turns > 40], f[turns > 40])
    assert torch.allclose(got[turns < 0.8], f[turns < 0.8] / factor, rtol=1e-15)
    ratio = got / f
    assert bool((ratio[1:] <= ratio[:-1]).all()) and 0 < int(((ratio < 1) & (ratio > 1 / factor)).sum())


@pytest.mark.parametrize("kwargs", [
    dict(head_dim=0), dict(head_dim=127), dict(head_dim=128, rotary_dim=130),
    dict(head_dim=128, rotary_dim=63), dict(head_dim=128, layout="spiral"),
    dict(head_dim=128, scaling="log"), dict(head_dim=128, theta=1.0),
    dict(head_dim=128, factor=0.0), dict(head_dim=128, factor=float("inf")),
    dict(head_dim=2, scaling="ntk", factor=2.0), dict(head_dim=128, scaling="by_parts", factor=2.0),
    dict(head_dim=128, scaling="by_parts", factor=0.5, original_context=4096),
    dict(head_dim=128, scaling="by_parts", factor=2.0, original_context=4096, beta_fast=1.0,
         beta_slow=2.0)])
def test_embedding_refuses(kwargs):
    with pytest.raises(ValueError):
        rotary.RotaryEmbedding(**kwargs, device="cpu")


def _call(**over):
    emb = rotary.RotaryEmbedding(128, device="cpu")
    a = dict(query=torch.zeros(3, 4, 128, dtype=torch.float16),
             key=torch.zeros(3, 2, 128, dtype=torch.float16),
             positions=torch.zeros(3, dtype=torch.int32), out_query=None, out_key=None)
    a.update(over)
    return emb.rotate(**a)


@pytest.mark.parametrize("over,message", [
    (dict(query=torch.zeros(3, 4, 128, dtype=torch.float64)), "FP16, BF16 or FP32"),
    (dict(positions=torch.zeros(3)), "int32 or int64"),
    (dict(positions=torch.zeros(6, dtype=torch.int32)[::2]), "int32 or int64"),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), "position each"),
    (dict(key=torch.zeros(3, 2, 128)), "one type"),
    (dict(key=torch.zeros(3, 2, 64, dtype=torch.float16)), "rotary rows must be"),
    (dict(out_query=torch.zeros(3, 4, 128)), "shaped and typed"),
    (dict(query=torch.zeros(3, 128, 4, dtype=torch.float16).transpose(1, 2)), "contiguous"),
    (dict(out_query=torch.zeros(1, 4, 128, dtype=torch.float16).expand(3, 4, 128)), "overlap"),
    (dict(out_query=torch.zeros(3 * 512 + 512, dtype=torch.float16).as_strided((3, 4, 128), (100, 128, 1))),
     "overlap"),
    (dict(), "current CUDA device"),
])
def test_rotate_refuses(over, message):
    with pytest.raises(ValueError, match=message):
        _call(**over)


def test_in_place_is_all_or_nothing():
    q = torch.zeros(3, 4, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="together"):
        _call(query=q, out_query=q)


@pytest.mark.skipif(torch.cuda.is_available(), reason="host-only checks of the C entry point")
@pytest.mark.parametrize("over,code,message", [
    (dict(head_dim=16386, rotary_dim=128), 3, "16384 dims"), (dict(query_heads=65536), 3, "65535 heads"),
    (dict(query_heads=0), 1, "with a head"), (dict(rotary_dim=130), 1, "even number"),
    (dict(position_bytes=2), 1, "int32 or int64"), (dict(dtype=3), 1, "FP16, BF16 or FP32"),
    (dict(out_query=None), 1, "null tensor"), (dict(tokens=1 << 50), 3, "too many rows")])
def test_c_entry_point_refuses(over, code, message):
    a = dict(query=4096, query_token=512, query_head=128, query_heads=4, key=None, key_token=0, key_head=0,
             key_heads=0, out_query=4096, out_query_token=512, out_query_head=128, out_key=None,
             out_key_token=0, out_key_head=0, positions=4096, position_bytes=4, turns=4096,
             amplitude=1.0, tokens=3, head_dim=128, rotary_dim=128, interleaved=0, dtype=0, stream=None)
    a.update(over)
    assert _capi.library().pg_rotate(*a.values()) == code and message in _capi.last_error()


@pytest.mark.parametrize("r,theta,context,factor", [
    (64, 1.0e4, 65536, 4.0), (32, 1.0e4, 65536, 8.0), (128, 1.0e4, 131072, 2.0), (8, 100.0, 8192, 4.0)])
def test_by_parts_where_the_slowest_pair_turns_more_than_once(r, theta, context, factor):
    """A ramp that ends past the last pair keeps its slope: no pair is stretched by the
    whole factor, and each by its place between the pairs that turn 32 times and once."""
    f = rotary.frequencies(r, theta)
    turns = f * context / (2 * math.pi)
    assert turns[-1] > 1.0
    got = rotary.frequencies(r, theta, "by_parts", factor, context)
    assert bool((got * factor > f * 1.01).all())
    # from one pair to the next, turns fall by theta^(2 / r)
    ends = [r / 2 * math.log(context / (2 * math.pi * n), theta) for n in (32.0, 1.0)]
    low, high = max(0, math.floor(ends[0])), min(r - 1, math.ceil(ends[1]))
    assert high > r // 2 - 1
    for i in range(r // 2):
        share = min(1.0, max(0.0, (i - low) / (high - low)))
        assert math.isclose(float(got[i]), float(f[i]) * (1 - share + share / factor), rel_tol=1e-12)


@pytest.mark.parametrize("name", ["query", "key"])
def test_rows_with_a_gradient_are_refused(name):
    """The result would have no history: it is not computed, but for no_grad()."""
    heads = {"query": 4, "key": 2}[name]
    rows = torch.zeros(3, heads, 128, dtype=torch.float16, requires_grad=True)
    for x in (rows, rows * 2.0):
        with pytest.raises(ValueError, match="no gradient"):
            _call(**{name: x})
    with torch.no_grad(), pytest.raises(ValueError, match="current CUDA device"):
        _call(**{name: rows})
