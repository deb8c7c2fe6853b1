"""Eviction from a paged cache by accumulated attention weight, and the attention that accumulates it.

Next to keys and values the cache of a layer has a third tensor, ``weight_pages [pages, Hkv, page]`` in 32 bits: for every cached
token and key head the softmax weights that queries gave it, summed over the heads of a group and over the queries so far.

``weighed_attention``          causal attention of prompts, and what weight every token got from it
``weighed_attention_varlen``   the same over sequences packed along time
``weighed_token_attention``    attention of new tokens over the cache (a token a sequence is plain decoding), which adds to the weights
``evict_tokens``               keeps the tokens of the largest weights, for every key head its own, and leaves the pages of the others

A serving loop: the weights of a prompt go to its tokens' slots (``weight_pages[slots // page, :, slots % page] = weights``) when
``append_tokens`` puts its keys and values there; every step takes ``weighed_token_attention`` and ``append_tokens`` with the same
slots; when a sequence has become too long, ``evict_tokens`` copies what stays to fresh pages and its old ones are free again.  Keys
keep the rotary positions that they were turned by; a sequence's length is then no longer the position of its next token.
Inference only.  Kernels: csrc/attention_weights.cu, csrc/paged_weigh.cu, csrc/evict.cu.
"""

from __future__ import annotations

import operator

import torch
from torch.autograd import forward_ad

from . import _lib, _validate
from .attention import _check, _forward, _launches, _packed_bounds, _sequences
from .paged import _DTYPES, _check_fresh, _check_pages, _check_table

_MOST_ROWS = 256      # new tokens times heads of a group


def _refuse_gradients(what, *tensors):
    if torch.is_grad_enabled() and any(x.requires_grad for x in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or with detached inputs")


def _weighed(what, q, k, v, bounds, scale):
    if forward_ad._current_level >= 0:
        _validate.refuse_tangents(what, q, k, v)
    if _lib.KERNEL_EVENTS is None and getattr(q, "is_cuda", False):
        done = _lib.host().weighed_attention(q, k, v, bounds, scale)
        if done is not None:
            return done
    checked, scale = _check(q, k, v, bounds, scale)
    _refuse_gradients(what, q, k, v)
    q, k, v = (_validate.detached(x) for x in (q, k, v))
    out, statistics, _ = _forward(q, k, v, checked, scale, (0, 0), True)
    weights = torch.empty(k.shape[:3], device=k.device, dtype=torch.float32)
    if statistics is None:
        return out, weights
    host, n_seq, rows = _sequences(q, checked)
    sizes = (host, n_seq, rows, q.shape[2], k.shape[2])
    with torch.cuda.device(q.device):
        size = _lib.lib().gdn2_attention_weights_bytes(*sizes)
    if size < 0:
        _lib.check(int(size), "gdn2_attention_weights_bytes")
    scratch = torch.empty(size, device=q.device, dtype=torch.uint8)
    strides = _lib.int64s(*(s for x in (q, k) for s in _validate.head_strides(x)))
    _lib.call("gdn2_attention_weights", q.device, q.data_ptr(), k.data_ptr(), statistics.data_ptr(), weights.data_ptr(),
              scratch.data_ptr() if size else None, strides, *sizes, q.shape[3], _lib.dtype_code(q.dtype), scale,
              _lib.stream_ptr(q.device), kernels=(1 + (size > 0)) * _launches(checked))
    return out, weights


def weighed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``causal_attention``, and the weight that every token got: ``(output, weights)``.

    ``weights [B, T, Hkv]`` (fp32): the softmax weights that a token was given by itself and by the tokens behind it, summed over
    these and over the heads of a group.  They are formed from scores in 32 bits, by exponentials of which a quarter is good to
    7e-6.  A query that has a score of NaN or +inf makes the weights of the tokens that it sees NaN; values do not enter them.
    No gradients."""

    return _weighed("weighed_attention", q, k, v, None, scale)


def weighed_attention_varlen(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens,
    *,
    scale: float | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``weighed_attention`` over ``N`` sequences packed along time, as in ``causal_attention_varlen``."""

    return _weighed("weighed_attention_varlen", q, k, v, _packed_bounds(q, cu_seqlens), scale)


def _check_weights(weight_pages, k_pages):
    pages, page, kv_heads, _ = k_pages.shape
    if not isinstance(weight_pages, torch.Tensor):
        raise TypeError("weight_pages must be a torch.Tensor")
    if weight_pages.dtype != torch.float32:
        raise TypeError("weight_pages must use torch.float32")
    if weight_pages.device != k_pages.device:
        raise ValueError("all inputs must be CUDA tensors on the same device")
    if weight_pages.shape != (pages, kv_heads, page) or not weight_pages.is_contiguous():
        raise ValueError(f"weight_pages must be contiguous with shape [{pages}, {kv_heads}, {page}]")


def _check_writes(writes, reads):
    """The ``writes``, contiguous tensors by name, overlap neither each other nor another tensor."""

    spans = {name: _validate.byte_span(x) for name, x in writes.items()}
    for name, span in spans.items():
        others = [other for x, other in spans.items() if x != name] + [_validate.extent(x) for x in reads]
        if any(_validate.spans_overlap(span, other) for other in others):
            raise ValueError(f"{name} must not overlap another tensor")


def weighed_token_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    weight_pages: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    slots: torch.Tensor,
    *,
    decay: float = 1.0,
    scale: float | None = None,
) -> torch.Tensor:
    """``tree_attention`` of a chain of ``N`` new tokens a sequence, which adds what weight the tokens got to ``weight_pages``.

    ``q [B, N, Hq, D]``, ``k`` and ``v [B, N, Hkv, D]`` belong to the new tokens, which are not in the cache yet; up to 256 of
    them times the heads of a group.  A cached token's weight becomes ``decay`` times what it was plus what it got, from all new
    tokens and heads of a group (a ``decay`` of 0 does not read what it was).  A new token's own weight is put to its place in
    ``slots`` (int64 ``[B, N]``), the place that ``append_tokens`` puts its key and value to; no cached token may have it, and a
    negative one, or one behind the cache, leaves it out.  A page of a sequence must not be another one's too.
    ``page_table`` and ``lengths`` as in ``tree_attention``; where those make a sequence's output NaN its weights become NaN, but
    for a bad length only those of its new tokens.  Scores of NaN or +inf make their sequence's and key head's
    weights NaN; values do not enter them.

    The call's workspace has 4 bytes for every query head, new token and token that ``page_table`` has room for, however long the
    sequences are (64 sequences, 32 heads, room for 131072 tokens: 1.1 GB).  A table with more columns than the longest sequence
    needs is better passed as ``page_table[:, :needed]``.  Keys and values are read once for every 16 rows (new tokens times heads
    of a group)."""

    if forward_ad._current_level >= 0:
        _validate.refuse_tangents("weighed_token_attention", q, k, v, k_pages, v_pages, weight_pages)
    if _lib.KERNEL_EVENTS is None and getattr(q, "is_cuda", False):
        done = _lib.host().weighed_token_attention(q, k, v, k_pages, v_pages, weight_pages, page_table, lengths, slots, decay, scale)
        if done is not None:
            return done
    batch, tokens, heads, kv_heads, dim = _check_fresh(q, k, v)
    _check_pages(k_pages, v_pages, q.dtype, q.device, kv_heads, dim)
    if k_pages.data_ptr() % 16 or v_pages.data_ptr() % 16:
        raise ValueError("k_pages and v_pages must be 16-byte aligned")
    _check_weights(weight_pages, k_pages)
    _check_table(page_table, lengths, batch, q.device)
    if not isinstance(slots, torch.Tensor) or slots.dtype != torch.int64:
        raise TypeError("slots must be a torch.int64 tensor")
    if slots.device != q.device:
        raise ValueError("all inputs must be CUDA tensors on the same device")
    if slots.shape != (batch, tokens):
        raise ValueError("slots must have shape [B, N]")
    if tokens * (heads // kv_heads) > _MOST_ROWS:
        raise NotImplementedError(f"up to {_MOST_ROWS} new tokens times heads of a group")
    if not isinstance(decay, (int, float)) or not 0.0 <= decay <= 1.0:
        raise ValueError("decay must be a number from 0 to 1")
    _refuse_gradients("weighed_token_attention", q, k, v, k_pages, v_pages, weight_pages)
    _lib.require_b200(q.device)
    scale = _validate.float32_scale(scale, dim)
    _check_writes({"weight_pages": weight_pages}, (q, k, v, k_pages, v_pages, page_table, lengths, slots))
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    if tokens == 0:
        return out
    page_table = page_table if page_table.stride(1) == 1 else page_table.contiguous()
    lengths, slots = lengths.contiguous(), slots.contiguous()
    columns, page = page_table.shape[1], k_pages.shape[1]
    with torch.cuda.device(q.device):
        size = _lib.lib().gdn2_weighed_token_workspace_bytes(batch, tokens, heads, kv_heads, dim, page, columns)
    if size < 0:
        _lib.check(int(size), "gdn2_weighed_token_workspace_bytes")
    workspace = torch.empty(size, device=q.device, dtype=torch.uint8)
    strides = _lib.int64s(*(s for x in (q, k, v) for s in _validate.head_strides(x)))
    _lib.call("gdn2_weighed_token_attention", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pages.data_ptr(),
              v_pages.data_ptr(), weight_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), slots.data_ptr(),
              out.data_ptr(), workspace.data_ptr(), strides, page_table.stride(0) if batch > 1 else columns, batch, tokens, heads,
              kv_heads, dim, k_pages.shape[0], page, columns, float(decay), _lib.dtype_code(q.dtype), scale, _lib.stream_ptr(q.device),
              kernels=2)
    torch.autograd.graph.increment_version((weight_pages,))
    return out


def evict_tokens(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    weight_pages: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    new_table: torch.Tensor,
    keep: int,
    *,
    sinks: int = 0,
    recent: int = 0,
) -> torch.Tensor:
    """Copy of every sequence the ``keep`` tokens of the largest weights to the pages in ``new_table``; returns the new lengths.

    Every key head keeps tokens of its own, in their order; the first ``sinks`` and the last ``recent`` tokens of a sequence are
    among them (``sinks + recent <= keep``).  Of equal weights the earlier token's counts more, NaN counts more than any number.
    A sequence of no more than ``keep`` tokens keeps all.  Their keys, values and weights are copied: token ``j`` of those that
    stay to page ``new_table[b, j // page]`` at ``j % page``.  ``new_table`` (int32 ``[B, columns]``, room for ``keep``) names
    pages of the same cache that no sequence uses: neither ``page_table`` nor another row of it; what lies in the old pages stays
    as it was, so that sequences may share them.  A new page number outside the cache leaves its tokens out; a row of -1 passes a
    sequence by.  Keys and values are fp16, bf16 or fp32.  The new lengths (int32 ``[B]``) are the smaller of ``lengths`` and
    ``keep``, of a sequence that is passed by too: it is where it was, and its old length is the one to go on with.  They are -1,
    with nothing copied, where a length or a page number of ``page_table`` is none of the cache.  Like ``page_table``, ``lengths``
    and ``new_table`` they stay on the device."""

    if forward_ad._current_level >= 0:
        _validate.refuse_tangents("evict_tokens", k_pages, v_pages, weight_pages)
    sizes = []
    for name, value, least in (("keep", keep, 1), ("sinks", sinks, 0), ("recent", recent, 0)):
        try:
            value = operator.index(value) if not isinstance(value, (bool, torch.Tensor)) else None
        except TypeError:
            value = None
        if value is None:
            raise TypeError(f"{name} must be an int")
        if value < least:
            raise ValueError(f"{name} must be at least {least}")
        sizes.append(value)
    keep, sinks, recent = sizes
    if sinks + recent > keep:
        raise ValueError("sinks and recent tokens must not be more than keep")
    if _lib.KERNEL_EVENTS is None and getattr(k_pages, "is_cuda", False):
        done = _lib.host().evict_tokens(k_pages, v_pages, weight_pages, page_table, lengths, new_table, keep, sinks, recent)
        if done is not None:
            return done
    if not isinstance(k_pages, torch.Tensor):
        raise TypeError("k_pages must be a torch.Tensor")
    if k_pages.ndim != 4:
        raise ValueError("k_pages must have shape [pages, page, Hkv, D]")
    if k_pages.dtype not in _DTYPES:
        raise TypeError("k_pages and v_pages must both use torch.bfloat16, torch.float16 or torch.float32")
    if not k_pages.is_cuda:
        raise ValueError("all inputs must be CUDA tensors on the same device")
    pages, page, kv_heads, dim = k_pages.shape
    _check_pages(k_pages, v_pages, k_pages.dtype, k_pages.device, kv_heads, dim)
    _check_weights(weight_pages, k_pages)
    batch = lengths.shape[0] if isinstance(lengths, torch.Tensor) and lengths.ndim == 1 else -1
    _check_table(page_table, lengths, batch, k_pages.device)
    if batch == 0:
        raise ValueError("batch must be positive")
    if not isinstance(new_table, torch.Tensor) or new_table.dtype != torch.int32:
        raise TypeError("new_table must be a torch.int32 tensor")
    if new_table.device != k_pages.device:
        raise ValueError("all inputs must be CUDA tensors on the same device")
    if new_table.ndim != 2 or new_table.shape[0] != batch or new_table.shape[1] * page < keep:
        raise ValueError("new_table must have shape [B, columns] with room for keep tokens")
    _refuse_gradients("evict_tokens", k_pages, v_pages, weight_pages)
    _lib.require_b200(k_pages.device)
    writes = {"k_pages": k_pages, "v_pages": v_pages, "weight_pages": weight_pages}
    _check_writes(writes, (page_table, lengths, new_table))
    page_table, new_table = (x if x.stride(1) == 1 else x.contiguous() for x in (page_table, new_table))
    lengths = lengths.contiguous()
    new_lengths = torch.empty(batch, device=k_pages.device, dtype=torch.int32)
    size = _lib.lib().gdn2_evict_workspace_bytes(batch, kv_heads, keep)
    if size < 0:
        _lib.check(int(size), "gdn2_evict_workspace_bytes")
    workspace = torch.empty(size, device=k_pages.device, dtype=torch.uint8)
    _lib.call("gdn2_evict_tokens", k_pages.device, k_pages.data_ptr(), v_pages.data_ptr(), weight_pages.data_ptr(),
              page_table.data_ptr(), lengths.data_ptr(), new_table.data_ptr(), new_lengths.data_ptr(), workspace.data_ptr(),
              page_table.stride(0) if batch > 1 else page_table.shape[1], new_table.stride(0) if batch > 1 else new_table.shape[1],
              batch, pages, page, kv_heads, dim, page_table.shape[1], new_table.shape[1], keep, sinks, recent,
              _lib.dtype_code(k_pages.dtype), _lib.stream_ptr(k_pages.device), kernels=2)
    torch.autograd.graph.increment_version((k_pages, v_pages, weight_pages))
    return new_lengths


__all__ = ["weighed_attention", "weighed_attention_varlen", "weighed_token_attention", "evict_tokens"]
