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
_LENGTHS = "lengths must be contiguous int32 [B]"
_PENALTIES = "penalties must be contiguous float32 [B]"
_BIASES = "biases must be contiguous int32 or int64 tokens and float32 values [B, n]"


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
    ``logits``, but not otherwise overlap them.  Logits, penalties and biases that
    autograd follows are refused: there is no backward pass.  Returns ``out``."""
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None or logits.dim() != 2:
        raise ValueError("logits must be FP16, BF16 or float32 [B, V] rows")
    batch, vocab = shape = logits.shape
    row, one = logits.stride()
    if one != 1 and vocab > 1:
        raise ValueError("logits must be FP16, BF16 or float32 [B, V] rows")
    device, at = logits.get_device(), logits.data_ptr()
    if out is None:
        out = torch.empty_like(logits)
        if vocab > 1 and out.stride(1) != 1:
            out = torch.empty(shape, device=logits.device, dtype=logits.dtype)
    elif out.shape != shape or out.dtype != logits.dtype or vocab > 1 and out.stride(1) != 1 \
            or batch > 1 and out.stride(0) < vocab:
        raise ValueError("shaped logits must be rows like the logits")
    elif out.data_ptr() == at and out.stride() != (row, one):
        raise ValueError("logits shaped in place must keep their strides")
    elif out.get_device() != device:
        raise ValueError(_capi.DEVICE_ERROR)
    _capi.refuse_gradients(logits, repetition, frequency, presence, bias_values)
    rows = (batch,)
    token_bytes = capacity = history_row = 0
    history_at = lengths_at = prompts_at = None
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
        if history.get_device() != device:
            raise ValueError(_capi.DEVICE_ERROR)
        lengths_at = _capi.pointer(history_lengths, torch.int32, rows, device, _LENGTHS)
        if prompt_lengths is not None:
            prompts_at = _capi.pointer(prompt_lengths, torch.int32, rows, device, _LENGTHS)
        capacity, token_bytes = history.shape[1], history.element_size()
        history_at, history_row = history.data_ptr(), history.stride(0)
    repetition_at, frequency_at, presence_at = (
        None if t is None else _capi.pointer(t, torch.float32, rows, device, _PENALTIES)
        for t in (repetition, frequency, presence))
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias tokens and values go together")
    biases, tokens_at, values_at = 0, None, None
    if bias_tokens is not None:
        if bias_tokens.dtype not in _TOKENS or bias_tokens.dim() != 2 or bias_tokens.shape[0] != batch:
            raise ValueError(_BIASES)
        if history is not None and history.dtype != bias_tokens.dtype:
            raise ValueError("history and bias tokens must have one type")
        tokens_at = _capi.pointer(bias_tokens, bias_tokens.dtype, bias_tokens.shape, device, _BIASES)
        values_at = _capi.pointer(bias_values, torch.float32, bias_tokens.shape, device, _BIASES)
        biases, token_bytes = bias_tokens.shape[1], bias_tokens.element_size()
    allowed_at, allowed_row = None, 0
    if allowed is not None:
        if allowed.dtype is not torch.int32 or allowed.shape != (batch, (vocab + 31) // 32) \
                or allowed.shape[1] > 1 and allowed.stride(1) != 1:
            raise ValueError("allowed must be int32 [B, ceil(V / 32)] rows of bits")
        if allowed.get_device() != device:
            raise ValueError(_capi.DEVICE_ERROR)
        allowed_at, allowed_row = allowed.data_ptr(), allowed.stride(0)
    stream = _capi.launch_stream(device)
    if batch == 0 or vocab == 0:
        return out
    if capacity == 0:       # a history of no tokens has no address
        history_at = lengths_at = prompts_at = repetition_at = frequency_at = presence_at = None
    if biases == 0:
        tokens_at = values_at = None
    _capi.call("pg_shape_logits", at, row, out.data_ptr(), out.stride(0), dtype, batch, vocab,
               history_at, history_row, capacity, lengths_at, prompts_at, repetition_at, frequency_at,
               presence_at, tokens_at, values_at, biases, token_bytes, allowed_at, allowed_row,
               stream)
    return out
