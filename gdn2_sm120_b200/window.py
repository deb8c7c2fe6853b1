"""Attention with a sliding window and a few first tokens that stay visible (sinks), for layers whose memory of the past is bounded.

Token ``i`` of a sequence sees the ``window`` last tokens, itself among them (``i - window < j <= i``), and the first ``sinks``
ones as far as they are not behind it.

``window_attention``          a batch of equally long sequences
``window_attention_varlen``   sequences of any lengths packed along time

Both are differentiable and run on the kernels of causal attention (csrc/attention_fwd.cu, csrc/attention_bwd.cu), which pass over
the tiles that no row of theirs sees; what is said in attention.py about types, heads, roundings and values that are not finite
holds here, with tiles that the window's edge or the sinks' end crosses beside those on the diagonal.  A window that reaches over
the longest sequence is causal attention, bit for bit.
"""

from __future__ import annotations

import operator

import torch

from .attention import _attention, _packed_bounds

_MOST = 2 ** 30     # tokens are numbered with fewer


def _window(window, sinks):
    """``(window, sinks)`` as the library takes them."""

    sizes = []
    for name, value, least in (("window", window, 1), ("sinks", sinks, 0)):
        try:
            value = operator.index(value) if not isinstance(value, (bool, torch.Tensor)) else None
        except TypeError:
            value = None
        if value is None:
            raise TypeError(f"{name} must be an int")
        if value < least:
            raise ValueError(f"{name} must be at least {least}")
        sizes.append(min(value, _MOST))
    return tuple(sizes)


def window_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    window: int,
    *,
    sinks: int = 0,
    scale: float | None = None,
) -> torch.Tensor:
    """``causal_attention`` in which a token sees the ``window`` last tokens, itself among them, and the first ``sinks``."""

    return _attention(q, k, v, None, scale, _window(window, sinks))


def window_attention_varlen(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens,
    window: int,
    *,
    sinks: int = 0,
    scale: float | None = None,
) -> torch.Tensor:
    """``window_attention`` over ``N`` sequences packed along time, as in ``causal_attention_varlen``; the sinks are each
    sequence's own."""

    return _attention(q, k, v, _packed_bounds(q, cu_seqlens), scale, _window(window, sinks))


__all__ = ["window_attention", "window_attention_varlen"]
