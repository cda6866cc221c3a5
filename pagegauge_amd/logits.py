"""Shaping of a step's logits before a token is picked from them.

``shape_logits`` applies the penalties for tokens a request has already seen,
its biases and the mask of the tokens its grammar allows, in one HIP launch
(``pg_shape_logits``); ``decoder.argmax_rows`` then picks the greedy token.
Lengths, tokens and penalties are read on the device, so a captured step sees
what the caller has written into them since.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _capi

_DTYPES = {torch.float16: _capi.PG_DTYPE_FP16, torch.bfloat16: _capi.PG_DTYPE_BF16,
           torch.float32: _capi.PG_DTYPE_FP32}
_TOKENS = (torch.int32, torch.int64)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def shape_logits(logits: torch.Tensor, out: Optional[torch.Tensor] = None, *,
                 history: Optional[torch.Tensor] = None,
                 history_lengths: Optional[torch.Tensor] = None,
                 prompt_lengths: Optional[torch.Tensor] = None,
                 repetition: Optional[torch.Tensor] = None,
                 frequency: Optional[torch.Tensor] = None,
                 presence: Optional[torch.Tensor] = None,
                 bias_tokens: Optional[torch.Tensor] = None,
                 bias_values: Optional[torch.Tensor] = None,
                 allowed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``logits`` [B, V] (FP16, BF16 or float32 rows) with, in this order and
    each where given:

    * ``repetition`` [B]: logits of tokens in ``history[b, :history_lengths[b]]``
      are divided by it where positive and multiplied by it elsewhere;
    * ``frequency`` and ``presence`` [B]: minus ``frequency`` times the count of
      the token in ``history[b, prompt_lengths[b]:history_lengths[b]]``, minus
      ``presence`` where it occurs there (without ``prompt_lengths``, in the
      whole history);
    * ``bias_values`` [B, n] added to the logits of ``bias_tokens`` [B, n] (of
      a token listed twice the last bias counts);
    * -inf for the tokens whose bit ``t % 32`` of ``allowed[b, t // 32]`` (int32)
      is clear, whatever their logit.

    ``history`` is int32 or int64 [B, capacity], each row's tokens first;
    lengths are int32 [B], the penalties and biases float32.  Tokens outside
    the vocabulary (padding) are ignored.  Computed in float32; ``out`` may be
    ``logits``.  Returns ``out``."""
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None or logits.dim() != 2 or logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("logits must be FP16, BF16 or float32 [B, V] rows")
    batch, vocab = logits.shape
    if out is None:
        out = torch.empty_like(logits)
        if vocab > 1 and out.stride(1) != 1:
            out = torch.empty((batch, vocab), device=logits.device, dtype=logits.dtype)
    elif out.shape != logits.shape or out.dtype != logits.dtype or vocab > 1 and out.stride(1) != 1 \
            or batch > 1 and out.stride(0) < vocab:
        raise ValueError("shaped logits must be rows like the logits")
    elif out.data_ptr() == logits.data_ptr() and out.stride() != logits.stride():
        raise ValueError("logits shaped in place must keep their strides")
    if history is None:
        if history_lengths is not None or prompt_lengths is not None or repetition is not None \
                or frequency is not None or presence is not None:
            raise ValueError("lengths and penalties need a history")
    else:
        if history.dtype not in _TOKENS or history.dim() != 2 or history.shape[0] != batch \
                or history.shape[1] > 1 and history.stride(1) != 1:
            raise ValueError("history must be int32 or int64 [B, capacity] rows")
        if history_lengths is None:
            raise ValueError("a history needs its lengths")
    for t in (history_lengths, prompt_lengths):
        if t is not None and (t.dtype is not torch.int32 or t.shape != (batch,) or not t.is_contiguous()):
            raise ValueError("lengths must be contiguous int32 [B]")
    for t in (repetition, frequency, presence):
        if t is not None and (t.dtype is not torch.float32 or t.shape != (batch,)
                              or not t.is_contiguous()):
            raise ValueError("penalties must be contiguous float32 [B]")
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias tokens and values go together")
    biases = 0
    if bias_tokens is not None:
        if bias_tokens.dtype not in _TOKENS or bias_tokens.dim() != 2 or bias_tokens.shape[0] != batch \
                or bias_values.shape != bias_tokens.shape or bias_values.dtype != torch.float32 \
                or not bias_tokens.is_contiguous() or not bias_values.is_contiguous():
            raise ValueError("biases must be int32 or int64 tokens and float32 values [B, n]")
        if history is not None and history.dtype != bias_tokens.dtype:
            raise ValueError("history and bias tokens must have one type")
        biases = bias_tokens.shape[1]
    if allowed is not None and (allowed.dtype != torch.int32 or allowed.dim() != 2
                                or allowed.shape != (batch, (vocab + 31) // 32)
                                or allowed.shape[1] > 1 and allowed.stride(1) != 1):
        raise ValueError("allowed must be int32 [B, ceil(V / 32)] rows of bits")
    _capi.require_current_device(logits, out, history, history_lengths, prompt_lengths, repetition,
                                 frequency, presence, bias_tokens, bias_values, allowed)
    if batch == 0 or vocab == 0:
        return out
    tokens = history if history is not None else bias_tokens
    # a history of no tokens has no address
    with_history = history is not None and history.shape[1] > 0
    _capi.call("pg_shape_logits", logits.data_ptr(), logits.stride(0), out.data_ptr(), out.stride(0),
               dtype, batch, vocab, history.data_ptr() if with_history else None,
               history.stride(0) if with_history else 0, history.shape[1] if with_history else 0,
               _ptr(history_lengths) if with_history else None,
               _ptr(prompt_lengths) if with_history else None,
               _ptr(repetition) if with_history else None, _ptr(frequency) if with_history else None,
               _ptr(presence) if with_history else None,
               _ptr(bias_tokens) if biases else None, _ptr(bias_values) if biases else None, biases,
               0 if tokens is None else tokens.element_size(), _ptr(allowed),
               0 if allowed is None else allowed.stride(0), _capi.current_stream())
    return out
