"""What ``shape_logits`` refuses, on the CPU."""

from __future__ import annotations

import pytest
import torch

from pagegauge_amd import _capi
from pagegauge_amd.logits import shape_logits

_F = torch.zeros(2)
_N = torch.zeros(2, dtype=torch.int32)
_H = torch.zeros(2, 5, dtype=torch.int64)


@pytest.mark.parametrize("logits,over,message", [
    (torch.zeros(2, 40, dtype=torch.float64), {}, "FP16, BF16 or float32"),
    (torch.zeros(40), {}, r"\[B, V\]"),
    (torch.zeros(40, 2).t(), {}, r"\[B, V\]"),
    (None, dict(out=torch.zeros(2, 41)), "rows like"),
    (None, dict(out=torch.zeros(1, 40).expand(2, 40)), "rows like"),
    (None, dict(repetition=_F), "need a history"),
    (None, dict(history_lengths=_N), "need a history"),
    (None, dict(history=_H), "needs its lengths"),
    (None, dict(history=_H.float(), history_lengths=_N), "int32 or int64"),
    (None, dict(history=_H[:1], history_lengths=_N), "int32 or int64"),
    (None, dict(history=_H, history_lengths=_N.long()), "lengths must be contiguous int32"),
    (None, dict(history=_H, history_lengths=_N, presence=_F.double()), "penalties must be contiguous float32"),
    (None, dict(history=_H, history_lengths=_N, frequency=torch.zeros(3)), "penalties must be contiguous float32"),
    (None, dict(bias_tokens=_H), "go together"),
    (None, dict(bias_tokens=_H, bias_values=torch.zeros(2, 4)), "biases must be"),
    (None, dict(history=_H.int(), history_lengths=_N, bias_tokens=_H, bias_values=torch.zeros(2, 5)),
     "one type"),
    (None, dict(allowed=torch.zeros(2, 1, dtype=torch.int32)), "allowed must be"),
    (None, dict(allowed=torch.zeros(2, 2, dtype=torch.int64)), "allowed must be"),
    (None, {}, "current CUDA device"),
])
def test_refusals(logits, over, message):
    with pytest.raises(ValueError, match=message):
        shape_logits(torch.zeros(2, 40) if logits is None else logits, **over)


@pytest.mark.skipif(torch.cuda.is_available(), reason="host-only checks of the C entry point")
@pytest.mark.parametrize("over,code,message", [
    (dict(logits=None), 1, "null tensor"), (dict(vocab=0), 1, "must be positive"),
    (dict(batch=70000), 3, "65535 rows"), (dict(dtype=3), 1, "FP16, BF16 or FP32"),
    (dict(history=4096), 1, "lengths"), (dict(presence=4096), 1, "need a history"),
    (dict(biases=1), 1, "go together"), (dict(history=4096, lengths=4096, capacity=1 << 30), 3, "2^30"),
    (dict(biases=1, bias_tokens=4096, bias_values=4096, token_bytes=2), 1, "int32 or int64")])
def test_c_entry_point_refuses(over, code, message):
    a = dict(logits=4096, logits_stride=32, out=4096, out_stride=32, dtype=2, batch=1, vocab=32,
             history=None, history_stride=0, capacity=0, lengths=None, prompts=None, repetition=None,
             frequency=None, presence=None, bias_tokens=None, bias_values=None, biases=0, token_bytes=8,
             allowed=None, allowed_stride=0, stream=None)
    a.update(over)
    assert _capi.library().pg_shape_logits(*a.values()) == code and message in _capi.last_error()


@pytest.mark.parametrize("name", ["logits", "repetition", "frequency", "presence", "bias_values"])
def test_gradients_are_refused(name):
    """The result would have no history: it is not computed, but for no_grad()."""
    a = dict(logits=torch.zeros(2, 40), history=_H, history_lengths=_N, repetition=_F, frequency=_F,
             presence=_F, bias_tokens=_H, bias_values=torch.zeros(2, 5))
    a[name] = a[name].clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        shape_logits(a.pop("logits"), **a)
