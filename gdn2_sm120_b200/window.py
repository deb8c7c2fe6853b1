"""Attention with a sliding window and a few first tokens that stay visible (sinks), for layers whose memory of the past is bounded.

Token ``i`` of a sequence sees the ``window`` last tokens, itself among them (``i - window < j <= i``), and the first ``sinks``
ones as far as they are not behind it.

``window_attention``          a batch of equally long sequences
``window_attention_varlen``   sequences of any lengths packed along time
``window_tree_attention``     drafted tokens, or single ones, over a paged cache, of which the window and the sinks are read

The first two are differentiable and run on the kernels of causal attention (csrc/attention_fwd.cu, csrc/attention_bwd.cu), which
pass over the tiles that no row of theirs sees.  What is said in attention.py about types, heads, roundings and values that are
not finite holds here, with tiles that the window's edge or the sinks' end crosses beside those on the diagonal.  Delta alone is
taken more exactly: from the output and what its rounding left over, which is kept for the backward.  A window that reaches over
the longest sequence is causal attention, bit for bit; but there, too, the gradients of sequences of at most 128 tokens have
delta with what rounding left over, whatever they are packed with.
"""

from __future__ import annotations

import operator

import torch

from .attention import _attention, _packed_bounds
from .paged import _tree_attention

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


def window_tree_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    window: int,
    mask: torch.Tensor | None = None,
    depths: torch.Tensor | None = None,
    *,
    sinks: int = 0,
    scale: float | None = None,
) -> torch.Tensor:
    """``tree_attention`` in which a drafted token sees the ``window`` last places, its own among them, and the first ``sinks``.

    A drafted token's place is ``lengths[b]`` plus its depth in the tree: ``depths`` (int32, ``[B, N]`` or ``[N]``, on the
    device; negative ones count as 0), which a ``mask`` needs; a chain (``mask=None``) has depths of ``0 .. N - 1`` where none
    are given.  Of the tokens that it would see without a window it sees those that lie less than ``window`` places before it,
    or on one of the first ``sinks`` places.  Pages that hold nothing but cached tokens that no drafted one sees are not read, so
    that they, and their entries in ``page_table``, may be anything.  Inference only."""

    return _tree_attention("window_tree_attention", q, k, v, k_pages, v_pages, page_table, lengths, mask, depths, _window(window, sinks), scale)


__all__ = ["window_attention", "window_attention_varlen", "window_tree_attention"]
