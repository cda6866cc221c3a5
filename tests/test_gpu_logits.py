"""``shape_logits`` against the same steps in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _want(logits, history, lengths, prompts, repetition, frequency, presence, bias_tokens, bias_values,
          allowed):
    """(shaped logits, size of the terms) in float64, token by token."""
    x = logits.double().cpu()
    batch, vocab = x.shape
    size = x.abs()
    for b in range(batch):
        tokens = [] if history is None else history[b, :max(0, int(lengths[b]))].tolist()
        made = tokens[max(0, int(prompts[b])) if prompts is not None else 0:]
        for t in {t for t in tokens if 0 <= t < vocab}:
            r = 1.0 if repetition is None else float(repetition[b])
            x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
            c = made.count(t)
            often = (0.0 if frequency is None else float(frequency[b])) * c
            once = 0.0 if presence is None or not c else float(presence[b])
            x[b, t] -= often + once
            # the two are taken off one after the other: x r - often, which is
            # rounded, may be as large as both though often + once is small
            # (0.1 - 0.12), so that each term counts by its own size
            size[b, t] = max(size[b, t], size[b, t] * r, size[b, t] / r) + abs(often) + abs(once)
        if bias_tokens is not None:
            for t, v in {int(t): float(v) for t, v in zip(bias_tokens[b], bias_values[b])}.items():
                if 0 <= t < vocab:
                    x[b, t] += v
                    size[b, t] += abs(v)
    if allowed is not None:
        token = torch.arange(vocab)
        bit = (allowed.cpu().long()[:, token // 32] >> (token % 32)) & 1
        x[bit == 0] = -math.inf
    return x, size


def _check(got, want, size):
    """Five float32 roundings of terms of that size, then half a step of the type."""
    eps = torch.finfo(got.dtype).eps
    got = got.double().cpu()
    masked = torch.isneginf(want)
    assert torch.equal(torch.isneginf(got), masked)
    allowed = size * 5 * 2.0 ** -24 + (want.abs() * eps / 2 * (1 + eps) if eps > 2.0 ** -20 else 0) + (
        2.0 ** -25 if eps == 2.0 ** -10 else 0)
    assert ((got - want).abs() <= allowed)[~masked].all()


def _case(cuda, batch, vocab, capacity, biases, dtype, token_type, seed=1):
    gen = torch.Generator().manual_seed(seed)
    a = dict(history=torch.randint(-3, vocab + 3, (batch, capacity), generator=gen),
             lengths=torch.randint(0, capacity + 1, (batch,), generator=gen).int())
    a["history"][:, ::2] = a["history"][:, ::2] % 7            # recurring tokens
    a["prompts"] = a["lengths"] // 3
    a["repetition"] = torch.rand(batch, generator=gen) + 0.6
    a["frequency"] = torch.rand(batch, generator=gen)
    a["presence"] = torch.rand(batch, generator=gen) - 0.3
    a["bias_tokens"] = torch.randint(-1, vocab + 1, (batch, biases), generator=gen)
    a["bias_values"] = torch.randn(batch, biases, generator=gen)
    a["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (batch, -(-vocab // 32)), generator=gen).int()
    logits = (torch.randn(batch, vocab, generator=gen) * 4).to(dtype)
    for n in ("history", "bias_tokens"):
        a[n] = a[n].to(token_type)
    return logits.to(cuda), {n: t.to(cuda) for n, t in a.items()}


def _run(logits, a, out=None):
    from pagegauge_amd.logits import shape_logits

    return shape_logits(logits, out, history=a["history"], history_lengths=a["lengths"],
                        prompt_lengths=a["prompts"], repetition=a["repetition"],
                        frequency=a["frequency"], presence=a["presence"],
                        bias_tokens=a["bias_tokens"], bias_values=a["bias_values"],
                        allowed=a["allowed"])


# tiles of every size, vocabularies that end inside a vector, a word and a tile; rows
# that start anywhere in a vector, and past the end of their last whole tile for it
@pytest.mark.parametrize("batch,vocab,capacity", [(1, 1, 1), (2, 31, 9), (3, 1000, 50), (1, 32768, 5000),
                                                  (5, 8197, 2), (130, 8192, 40), (9, 2047, 20),
                                                  (9, 50001, 700), (300, 3, 4), (300, 2047, 20),
                                                  (257, 8191, 3), (90, 10241, 30)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("token_type", [torch.int32, torch.int64])
def test_all_parts(cuda, batch, vocab, capacity, dtype, token_type):
    print(f"logits {batch} x {vocab} history {capacity} {dtype} {token_type}", flush=True)
    logits, a = _case(cuda, batch, vocab, capacity, 6, dtype, token_type)
    got = _run(logits, a)
    _check(got, *_want(logits, **a))
    again = logits.clone()
    assert _run(again, a, again) is again
    assert torch.equal(again.view(torch.uint8), got.view(torch.uint8))


@pytest.mark.parametrize("given", [(), ("allowed",), ("bias",), ("repetition",), ("frequency",),
                                   ("presence", "allowed"), ("history",)])
def test_parts_left_out(cuda, given):
    from pagegauge_amd.logits import shape_logits

    logits, a = _case(cuda, 3, 3001, 64, 5, torch.float32, torch.int64)
    kept = {n: None for n in ("repetition", "frequency", "presence", "bias_tokens", "bias_values",
                              "allowed", "prompts")}
    names = [x for n in given for x in (("bias_tokens", "bias_values") if n == "bias" else (n,))]
    kept.update({n: a[n] for n in names if n in kept})
    history = any(n in names for n in ("repetition", "frequency", "presence", "history"))
    got = shape_logits(logits, history=a["history"] if history else None,
                       history_lengths=a["lengths"] if history else None,
                       repetition=kept["repetition"], frequency=kept["frequency"],
                       presence=kept["presence"], bias_tokens=kept["bias_tokens"],
                       bias_values=kept["bias_values"], allowed=kept["allowed"])
    want = _want(logits, a["history"] if history else None, a["lengths"], **kept)
    _check(got, *want)
    if given in ((), ("history",)):
        assert torch.equal(got, logits)


def test_strides_alignment_and_padding(cuda):
    """Rows of a wider buffer, unaligned rows, and lengths outside the capacity."""
    logits, a = _case(cuda, 4, 777, 30, 3, torch.float32, torch.int32)
    a["lengths"] = torch.tensor([-5, 0, 30, 1000], device=cuda, dtype=torch.int32)
    a["prompts"] = torch.tensor([0, 7, -2, 40], device=cuda, dtype=torch.int32)
    want = _want(logits, **a)
    _check(_run(logits, a), *want)
    for width, begin in ((784, 0), (781, 3)):
        wide = torch.full((4, width), 5.0, device=cuda)
        wide[:, begin:begin + 777] = logits
        hist = torch.full((4, 41), 3, device=cuda, dtype=torch.int32)
        hist[:, 2:32] = a["history"]
        b = dict(a, history=hist[:, 2:32])
        view = wide[:, begin:begin + 777]
        _run(view, b, view)
        _check(view, *want)
        assert (wide[:, :begin] == 5.0).all() and (wide[:, begin + 777:] == 5.0).all()
    # as many rows as make larger tiles, in rows of another buffer, whose ends are kept
    logits, a = _case(cuda, 270, 777, 30, 3, torch.float16, torch.int32)
    want = _want(logits, **a)
    for width, begin in ((784, 0), (789, 5)):
        wide = torch.full((270, width), 5.0, device=cuda, dtype=torch.float16)
        wide[:, begin:begin + 777] = logits
        view = wide[:, begin:begin + 777]
        _run(view, a, view)
        _check(view, *want)
        assert (wide[:, :begin] == 5.0).all() and (wide[:, begin + 777:] == 5.0).all()
    # an output whose rows lie otherwise than the logits'
    logits, a = _case(cuda, 260, 777, 30, 3, torch.float32, torch.int32)
    want = _want(logits, **a)
    other = torch.full((260, 779), 5.0, device=cuda)
    _check(_run(logits, a, other[:, 1:778]), *want)
    assert (other[:, 0] == 5.0).all() and (other[:, 778] == 5.0).all()


def test_extreme_logits(cuda):
    """Infinities, NaN and zeros pass as the arithmetic has them; the mask wins;
    a request that may pick nothing has -inf everywhere."""
    from pagegauge_amd.logits import shape_logits

    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[inf, -inf, nan, 0.0, -0.0, 1.0]] * 2, device=cuda)
    history = torch.arange(6, device=cuda).expand(2, 6)
    n = torch.tensor([6, 6], device=cuda, dtype=torch.int32)
    two = torch.full((2,), 2.0, device=cuda)
    got = shape_logits(logits, history=history, history_lengths=n, repetition=two, presence=two)
    assert got[0, :2].tolist() == [inf, -inf] and got[0, 2].isnan()
    assert got[0, 3:].tolist() == [-2.0, -2.0, -1.5]
    allowed = torch.tensor([[0b111000], [0]], device=cuda, dtype=torch.int32)
    got = shape_logits(logits, allowed=allowed)
    assert got[0].tolist() == [-inf, -inf, -inf, 0.0, 0.0, 1.0] and torch.isneginf(got[1]).all()
    empty = torch.empty(0, 100, device=cuda)
    assert shape_logits(empty).shape == (0, 100)
    none = torch.empty(2, 0, device=cuda, dtype=torch.int64)
    got = shape_logits(logits, history=none, history_lengths=n, repetition=two)
    assert torch.equal(got[:, 3:], logits[:, 3:])


def test_same_token_twice_is_deterministic(cuda):
    """A token of a long history counted exactly, the last of two biases kept."""
    from pagegauge_amd.logits import shape_logits

    logits = torch.zeros(1, 40, device=cuda)
    history = torch.full((1, 20000), 33, device=cuda, dtype=torch.int32)
    n = torch.tensor([20000], device=cuda, dtype=torch.int32)
    p = torch.tensor([1], device=cuda, dtype=torch.int32)
    one = torch.ones(1, device=cuda)
    tokens = torch.tensor([[5, 33, 5, -1, 40, 5]], device=cuda, dtype=torch.int32)
    values = torch.tensor([[1.0, 2.0, 4.0, 8.0, 16.0, 32.0]], device=cuda)
    got = shape_logits(logits, history=history, history_lengths=n, prompt_lengths=p, frequency=one,
                       bias_tokens=tokens, bias_values=values)
    want = torch.zeros(1, 40)
    want[0, 33], want[0, 5] = -19999.0 + 2.0, 32.0
    assert torch.equal(got.cpu(), want)


def test_captured_step_reads_what_was_written_since(cuda):
    """shape_logits and argmax_rows in one graph: each replay appends its token
    to the history, which the next one sees."""
    from pagegauge_amd.decoder import argmax_rows
    from pagegauge_amd.logits import shape_logits

    logits = torch.tensor([[3.0, 2.5, 2.0, 0.0], [0.0, 1.0, 1.5, 1.25]], device=cuda)
    history = torch.zeros(2, 8, device=cuda, dtype=torch.int64)
    n = torch.zeros(2, device=cuda, dtype=torch.int32)
    presence = torch.full((2,), 10.0, device=cuda)
    out, token = torch.empty_like(logits), torch.zeros(2, device=cuda, dtype=torch.int64)

    def step():
        shape_logits(logits, out, history=history, history_lengths=n, presence=presence)
        argmax_rows(out, token)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    picked = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        picked.append(token.tolist())
        history[:, i] = token
        n += 1
    assert picked == [[0, 2], [1, 3], [2, 1], [3, 0]]
