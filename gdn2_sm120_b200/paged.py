"""A paged cache of keys and values, and attention over it, for serving full-attention layers.

The cache of a layer is two contiguous tensors ``[pages, page, Hkv, D]``.  Which pages a sequence has is the caller's
business: a row of ``page_table`` names them, its cached token ``t`` lies in page ``page_table[b, t // page]`` at
``t % page``.

``append_tokens``    writes the keys and values of tokens to their slots
``tree_attention``   attention of drafted tokens over the cache and over their own ancestors; one token a sequence is
                     plain decoding

A step of speculative decoding: ``tree_attention`` with the drafts' keys and values beside the cache, then
``append_tokens`` with the slots of the accepted ones (-1 for the others).  Kernels: csrc/paged.cu,
csrc/paged_tiles.cuh, csrc/paged_tree.cuh.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib, _validate

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check_pages(k_pages, v_pages, dtype, device, kv_heads, dim):
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if x.ndim != 4 or x.shape[2:] != (kv_heads, dim):
            raise ValueError(f"{name} must have shape [pages, page, {kv_heads}, {dim}]")
        if x.dtype != dtype:
            raise TypeError(f"{name} must have the dtype of k and v")
        if x.device != device:
            raise ValueError("all inputs must be CUDA tensors on the same device")
        if not x.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if 0 in x.shape:
            raise ValueError(f"{name} must not be empty")
    if k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must have the same shape")


def append_tokens(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    slots: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Copy the keys and values of tokens into the cache; returns ``(k_pages, v_pages)``, which it changes.

    ``k`` and ``v`` are ``[N, Hkv, D]`` or ``[B, T, Hkv, D]``; ``slots`` (int64, ``[N]`` or ``[B, T]``) names each
    token's place, ``page number * page + place in the page``.  A slot that is negative or behind the cache leaves the
    token out.  Two tokens with one slot are not allowed (which of them stays is undefined).  fp16, bf16 or fp32.  Inference
    only."""

    if forward_ad._current_level >= 0:
        _validate.refuse_tangents("append_tokens", k, v, k_pages, v_pages)
    if _lib.KERNEL_EVENTS is None and getattr(k, "is_cuda", False):
        if _lib.host().append_tokens(k, v, k_pages, v_pages, slots):
            return k_pages, v_pages
    if not all(isinstance(x, torch.Tensor) for x in (k, v, slots)):
        raise TypeError("k, v, and slots must be torch.Tensor objects")
    if k.ndim not in (3, 4) or k.shape != v.shape:
        raise ValueError("k and v must have the same shape, [N, H, D] or [B, T, H, D]")
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise TypeError("k and v must both use torch.bfloat16, torch.float16 or torch.float32")
    if not k.is_cuda or any(x.device != k.device for x in (v, slots)):
        raise ValueError("all inputs must be CUDA tensors on the same device")
    if slots.shape != k.shape[:-2]:
        raise ValueError("slots must have one entry for every token")
    if slots.dtype != torch.int64:
        raise TypeError("slots must use torch.int64")
    heads, dim = k.shape[-2:]
    _check_pages(k_pages, v_pages, k.dtype, k.device, heads, dim)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise RuntimeError("append_tokens has no gradient: call it under torch.no_grad() or with detached inputs")
    _lib.require_b200(k.device)
    spans = [_validate.byte_span(x) for x in (k_pages, v_pages)]
    if _validate.spans_overlap(*spans) or any(
            _validate.spans_overlap(_validate.extent(x), s) for x in (k, v, slots) for s in spans):
        raise ValueError("k_pages and v_pages must not overlap each other or another tensor")
    k, v, slots = (x.detach().reshape(-1, *x.shape[slots.ndim:]) for x in (k, v, slots))
    if k.shape[0] == 0:
        return k_pages, v_pages
    k, v = (x if x.stride(2) == 1 else x.contiguous() for x in (k, v))
    slots = slots.contiguous()
    strides = _lib.int64s(k.stride(0), k.stride(1), v.stride(0), v.stride(1))
    _lib.call("gdn2_append_tokens", k.device, k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
              slots.data_ptr(), strides, k.shape[0], k_pages.shape[0], k_pages.shape[1], heads, dim,
              _lib.dtype_code(k.dtype), _lib.stream_ptr(k.device))
    torch.autograd.graph.increment_version((k_pages, v_pages))     # a backward that has saved them must not use them any more
    return k_pages, v_pages


def tree_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    mask: torch.Tensor | None = None,
    *,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of ``N`` drafted tokens of each sequence over its cache and over each other.

    ``q [B, N, Hq, D]``, ``k`` and ``v [B, N, Hkv, D]`` belong to the drafted tokens, which are not in the cache;
    fp16 or bf16, ``D`` a multiple of 8 up to 128.  Token ``i`` of sequence ``b`` sees the ``lengths[b]`` cached tokens
    and those drafted tokens ``j`` with ``mask[b, i, j]`` (bool, ``[B, N, N]`` or ``[N, N]``): itself and its ancestors
    in a tree.  ``mask=None`` is a chain, ``j <= i``.  A token that sees nothing gets 0.  What no token sees (the rest of
    a page, another branch) may hold anything.  ``page_table`` (int32 ``[B, columns]``) and ``lengths`` (int32 ``[B]``)
    stay on the device: no call waits for it, and a captured graph may be replayed with other contents.  A page number
    outside the cache or a length beyond ``columns`` pages makes the sequence's output NaN.  Inference only."""

    return _tree_attention("tree_attention", q, k, v, k_pages, v_pages, page_table, lengths, mask, None, (0, 0), scale)


def _check_table(page_table, lengths, batch, device):
    for name, x, dims in (("page_table", page_table, 2), ("lengths", lengths, 1)):
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if x.dtype != torch.int32:
            raise TypeError(f"{name} must use torch.int32")
        if x.device != device:
            raise ValueError("all inputs must be CUDA tensors on the same device")
        if x.ndim != dims or x.shape[0] != batch:
            raise ValueError("page_table must have shape [B, columns] and lengths [B]")
    if page_table.shape[1] == 0:
        raise ValueError("page_table must have a column")


def _check_fresh(q, k, v):
    """Queries, keys and values of tokens that are not in the cache: ``(batch, tokens, heads, kv_heads, dim)``."""

    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    for name, x in (("q", q), ("k", k), ("v", v)):
        _validate.heads_tensor(name, x, q.device, q.dtype)
    batch, tokens, heads, dim = q.shape
    if k.shape != v.shape or k.shape[:2] != (batch, tokens) or k.shape[3] != dim:
        raise ValueError("k and v must have the same shape, and q's [B, N] and D")
    kv_heads = k.shape[2]
    if min(batch, heads, kv_heads) <= 0:
        raise ValueError("batch and heads must be positive")
    if heads % kv_heads:
        raise ValueError("the number of query heads must be a multiple of that of key heads")
    return batch, tokens, heads, kv_heads, dim


def _tree_attention(what, q, k, v, k_pages, v_pages, page_table, lengths, mask, depths, window, scale):
    if forward_ad._current_level >= 0:
        _validate.refuse_tangents(what, q, k, v, k_pages, v_pages)
    if _lib.KERNEL_EVENTS is None and getattr(q, "is_cuda", False):
        done = _lib.host().tree_attention(q, k, v, k_pages, v_pages, page_table, lengths, mask, depths, *window, scale)
        if done is not None:
            return done
    batch, drafted, heads, kv_heads, dim = _check_fresh(q, k, v)
    _check_pages(k_pages, v_pages, q.dtype, q.device, kv_heads, dim)
    if k_pages.data_ptr() % 16 or v_pages.data_ptr() % 16:
        raise ValueError("k_pages and v_pages must be 16-byte aligned")
    _check_table(page_table, lengths, batch, q.device)
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool:
            raise TypeError("mask must be a torch.bool tensor or None")
        if mask.device != q.device:
            raise ValueError("all inputs must be CUDA tensors on the same device")
        if mask.shape not in ((drafted, drafted), (batch, drafted, drafted)):
            raise ValueError("mask must have shape [B, N, N] or [N, N]")
    if depths is not None:
        if not isinstance(depths, torch.Tensor) or depths.dtype != torch.int32:
            raise TypeError("depths must be a torch.int32 tensor or None")
        if depths.device != q.device:
            raise ValueError("all inputs must be CUDA tensors on the same device")
        if depths.shape not in ((drafted,), (batch, drafted)):
            raise ValueError("depths must have shape [B, N] or [N]")
    elif mask is not None and window != (0, 0):
        raise ValueError("a mask needs the depths of the drafted tokens")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or with detached inputs")
    _lib.require_b200(q.device)
    scale = _validate.float32_scale(scale, dim)
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    if drafted == 0:
        return out
    q, k, v = (_validate.detached(x) for x in (q, k, v))
    page_table = page_table if page_table.stride(1) == 1 else page_table.contiguous()
    lengths = lengths.contiguous()
    if mask is not None:
        mask = mask.contiguous()
    more = ((), (), ())
    if window != (0, 0):
        depths = depths if depths is None else depths.contiguous()
        more = ((_lib.ptr(depths),), (0 if depths is None or depths.ndim == 1 else drafted,), window)
    with torch.cuda.device(q.device):
        size = _lib.lib().gdn2_tree_workspace_bytes(drafted, heads, kv_heads, dim)
    if size < 0:
        _lib.check(int(size), "gdn2_tree_workspace_bytes")
    workspace = torch.empty(size, device=q.device, dtype=torch.uint8)
    strides = _lib.int64s(*(s for x in (q, k, v) for s in _validate.head_strides(x)))
    _lib.call(f"gdn2_{what}", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pages.data_ptr(),
              v_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), _lib.ptr(mask), *more[0], out.data_ptr(),
              workspace.data_ptr(), strides, page_table.stride(0) if batch > 1 else page_table.shape[1],
              0 if mask is None or mask.ndim == 2 else drafted * drafted, *more[1], batch, drafted, heads, kv_heads, dim,
              k_pages.shape[0], k_pages.shape[1], page_table.shape[1], *more[2], _lib.dtype_code(q.dtype), scale,
              _lib.stream_ptr(q.device), kernels=2)
    return out


__all__ = ["append_tokens", "tree_attention"]
