"""Causal attention with a sliding window and sinks: training, prefill and
single tokens against a cache."""
from __future__ import annotations

from typing import Optional

import torch

from . import ext


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                     lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v over the keys that a row sees; [B, T, H, D].

    q is [B, T, H, D], k and v are [B, T, Hkv, D]; H / Hkv query heads share a
    key head.  Row i of sequence b sees key j iff ``i < lengths[b]``,
    ``j <= i`` and (``i - j < window`` or ``j < sinks``): the last ``window``
    tokens, itself among them, and the first ``sinks``.  A window of T or more
    is full causal attention.  ``lengths`` (int32 [B], on the device, clamped to
    [0, T]) are the sequences' lengths; rows at or behind them give zeros and
    get zero gradients, and what they hold is not used.  Inside a sequence a
    value that is not finite may reach rows that do not see it, as in a matrix
    product with zeros.  ``scale`` is D ** -0.5 unless given.

    float32, bfloat16 or float16, D from 1 to 128, any strides (elements of a
    head that do not lie side by side are copied first).  Scores, softmax
    statistics and sums are 32-bit.  With 16-bit inputs of more than 64 tokens
    the probabilities, and in the backward pass their gradients, are rounded to
    the input type where they enter a matrix product; rows of few keys (the
    first 128, or all where window + sinks <= 128 or D < 64) keep twice the bits
    of the probabilities.  float16 scales those gradients by a bound of their
    own size, row by row and key by key, so nothing overflows before the result
    does; what lies 2^29 below that bound loses bits.  A row whose scores are all
    minus infinity gives zeros.

    Gradients flow to q, k and v, each summed in a fixed order: the same inputs
    give the same bits.  A kernel that waits in vain for its data (two seconds)
    gives up, and the next call on the device raises RuntimeError.
    """
    return ext.get_ops().window_attention(q, k, v, window, sinks, lengths, scale)


def window_attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, window: int,
                            sinks: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """One token per sequence against a cache; [B, H, D].

    q is [B, H, D], the caches are [B, T, Hkv, D] and already hold the token's
    own key and value: the query is token ``lengths[b] - 1`` of its sequence and
    sees what that row of ``window_attention`` sees.  ``lengths`` (int32 [B], on
    the device) are clamped to [0, T]; a length of 0 gives zeros.  Only the keys
    and values that are seen are used.  Everything is 32-bit but the result's
    own rounding (16-bit caches: p is kept to twice the type's bits).  No
    backward pass.
    """
    return ext.get_ops().window_attention_decode(q, k_cache, v_cache, lengths, window, sinks, scale)
