"""Rotary positions from 64-bit angles, for contexts of any length.

``RotaryEmbedding`` holds the frequencies of one model; ``rotate`` turns the
query and key rows of any tokens in one HIP launch (``pg_rotate``): pairs of
the two halves of the rotated part (``"half"``, the layout of ``decoder.rope``)
or neighbouring dims (``"interleaved"``), the whole head or its first
``rotary_dim`` dims, and frequencies scaled for contexts longer than the model
was trained on:

* ``"linear"``: positions divided by ``factor``;
* ``"ntk"``: the base raised to ``theta * factor^(R / (R - 2))``, which keeps the
  fastest pair and stretches the slowest by ``factor``;
* ``"by_parts"``: pairs that turn more than ``beta_fast`` times within
  ``original_context`` keep their frequency, those that turn less than
  ``beta_slow`` times are divided by ``factor``, with a linear ramp over the
  pairs between (its ends rounded outwards to whole pairs, within 0 and
  ``rotary_dim - 1``), and both rows scaled by ``0.1 ln(factor) + 1`` (unless
  ``attention_factor`` is given).

The angles are worked out in the kernel, so nothing grows with the context; they
are good to 2^-22 of a turn at position 2^31 (and to 2^-51 of themselves beyond);
``int4.rope_append`` uses the same object.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _capi

_DTYPES = {torch.float16: _capi.PG_DTYPE_FP16, torch.bfloat16: _capi.PG_DTYPE_BF16,
           torch.float32: _capi.PG_DTYPE_FP32}
_POSITIONS = (torch.int32, torch.int64)
_NO_ROWS = (None, 0, 0, 0, None, 0, 0)
LAYOUTS = ("half", "interleaved")
SCALINGS = ("none", "linear", "ntk", "by_parts")


def frequencies(rotary_dim: int, theta: float, scaling: str = "none", factor: float = 1.0,
                original_context: Optional[int] = None, beta_fast: float = 32.0,
                beta_slow: float = 1.0) -> torch.Tensor:
    """Radians per position of each of the ``rotary_dim / 2`` pairs (float64, CPU)."""
    r = rotary_dim
    if scaling == "ntk":
        theta = theta * factor ** (r / (r - 2))
    f = theta ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if scaling == "linear":
        return f / factor
    if scaling != "by_parts":
        return f

    def pair(turns: float) -> float:     # the pair that turns so many times
        return r * math.log(original_context / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

    # the ramp may end past the last of the r / 2 pairs, whose frequencies it then does not
    # stretch by the whole factor
    low = max(math.floor(pair(beta_fast)), 0)
    high = min(math.ceil(pair(beta_slow)), r - 1)
    ramp = ((torch.arange(r // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1.0 - ramp) + f / factor * ramp


class RotaryEmbedding:
    """Frequencies, layout and amplitude of a model's rotary positions."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, theta: float = 1.0e6,
                 layout: str = "half", scaling: str = "none", factor: float = 1.0,
                 original_context: Optional[int] = None, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attention_factor: Optional[float] = None,
                 device="cuda") -> None:
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim <= 0 or head_dim % 2 or rotary_dim <= 0 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError("the rotated part must be an even number of a head's dims")
        if layout not in LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout}")
        if scaling not in SCALINGS:
            raise ValueError(f"unknown rotary scaling {scaling}")
        if not (theta > 1.0 and math.isfinite(theta)) or not (factor > 0.0 and math.isfinite(factor)):
            raise ValueError("theta must exceed 1 and the factor be positive, both finite")
        if attention_factor is not None and not math.isfinite(attention_factor):
            raise ValueError("the attention factor must be finite")
        if scaling == "ntk" and rotary_dim < 4:
            raise ValueError("ntk scaling needs at least two pairs")
        if scaling == "by_parts" and (not original_context or original_context <= 0
                                      or not beta_fast >= beta_slow > 0 or factor < 1.0):
            raise ValueError("by_parts scaling needs the original context, a factor of at least 1 "
                             "and beta_fast >= beta_slow > 0")
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        f = frequencies(rotary_dim, theta, scaling, factor, original_context, beta_fast, beta_slow)
        self.turns = (f / (2.0 * math.pi)).to(device)
        if attention_factor is not None:
            self.amplitude = float(attention_factor)
        else:
            self.amplitude = 0.1 * math.log(factor) + 1.0 if scaling == "by_parts" else 1.0

    @property
    def interleaved(self) -> bool:
        return self.layout == "interleaved"

    def rotate(self, query: torch.Tensor, key: Optional[torch.Tensor], positions: torch.Tensor,
               out_query: Optional[torch.Tensor] = None, out_key: Optional[torch.Tensor] = None):
        """(rotated query, rotated key) of rows [T, H, head_dim] at ``positions``
        [T] (int32 or int64): FP16, BF16 or FP32, any token and head strides
        (slices of a fused projection).  ``key`` may be None.  The outputs may
        be the inputs themselves, but not otherwise overlap them.  Rows that
        autograd follows are refused: there is no backward pass."""
        dtype = _DTYPES.get(query.dtype)
        if dtype is None:
            raise ValueError("rotary rows must be FP16, BF16 or FP32")
        if positions.dim() != 1 or positions.dtype not in _POSITIONS or not positions.is_contiguous():
            raise ValueError("positions must be contiguous int32 or int64 [T]")
        tokens = positions.shape[0]
        out_query, query_args, in_place = self._rows(query, out_query, tokens, query.dtype)
        key_args = _NO_ROWS
        if key is not None:
            out_key, key_args, key_in_place = self._rows(key, out_key, tokens, query.dtype)
            if in_place != key_in_place:
                raise ValueError("query and key are rotated in place together or not at all")
        _capi.refuse_gradients(query, key)
        device = query.get_device()
        if positions.get_device() != device or self.turns.get_device() != device \
                or out_query.get_device() != device \
                or key is not None and (key.get_device() != device or out_key.get_device() != device):
            raise ValueError(_capi.DEVICE_ERROR)
        stream = _capi.launch_stream(device)
        if tokens and query_args[3] + key_args[3]:
            _capi.call("pg_rotate", *query_args[:4], *key_args[:4], *query_args[4:], *key_args[4:],
                       positions.data_ptr(), positions.element_size(), self.turns.data_ptr(),
                       self.amplitude, tokens, self.head_dim, self.rotary_dim,
                       int(self.interleaved), dtype, stream)
        return out_query, out_key

    def _rows(self, x: torch.Tensor, out: Optional[torch.Tensor], tokens: int, dtype):
        """(out, (x, token and head strides, heads, out, its strides), in place)."""
        shape = x.shape
        if len(shape) != 3 or shape[0] != tokens or shape[2] != self.head_dim or x.dtype != dtype:
            raise ValueError(f"rotary rows must be [T, H, {self.head_dim}] of one type, with a "
                             "position each")
        token, head, dim = x.stride()
        if dim != 1:
            raise ValueError("a head's dims must be contiguous")
        heads = shape[1]
        at = x.data_ptr()
        if out is None:
            out = torch.empty_like(x)
            if not out.is_contiguous():
                out = torch.empty(shape, device=x.device, dtype=dtype)
            return out, (at, token, head, heads, out.data_ptr(), heads * self.head_dim,
                         self.head_dim), False
        if out.shape != shape or out.dtype != dtype:
            raise ValueError("rotated rows must be shaped and typed like the rows")
        out_token, out_head, out_dim = out.stride()
        if out_dim != 1:
            raise ValueError("a head's dims must be contiguous")
        # the [T, H] rows of head_dim dims must lie apart
        (near, inner), (far, _) = sorted(((out_token, tokens), (out_head, heads)))
        if tokens > 1 and heads > 1:
            apart = near >= self.head_dim and far >= near * (inner - 1) + self.head_dim
        else:
            apart = tokens * heads <= 1 or (out_token if tokens > 1 else out_head) >= self.head_dim
        if not apart:
            raise ValueError("rotated rows must not overlap each other")
        in_place = out.data_ptr() == at
        if in_place and (out_token, out_head) != (token, head):
            raise ValueError("rows rotated in place must keep their strides")
        return out, (at, token, head, heads, out.data_ptr(), out_token, out_head), in_place
