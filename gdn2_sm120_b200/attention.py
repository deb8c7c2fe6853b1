"""Causal attention over whole sequences, for the full-attention layers between Gated DeltaNet-2 layers.

``causal_attention``          a batch of equally long sequences
``causal_attention_varlen``   sequences of any lengths packed along time, as in ``chunk_gdn2_varlen``

Both are differentiable and run on the tensor cores (csrc/attention_fwd.cu, csrc/attention_bwd.cu): scores, statistics and
sums are in 32 bits.  What goes into a product is rounded to the inputs' type, which is what the tensor cores take: the
weights P for their product with the values (exponentials are good to 2^-17), and in the backward P and the slopes dS = P (dP -
delta); delta_i = do_i . o_i is taken from the output as it was returned.  ``Hq`` query heads share ``Hkv`` key and value
heads in groups of ``Hq / Hkv`` consecutive ones; the gradients of a shared head are summed in 32 bits before they are rounded.

An output depends on what its row sees and on nothing else, whatever the tensors hold elsewhere.  Gradients do where q, k and the
cotangent are finite.  A key that is not also reaches dq, in its channel, of the rows before it in its tile of 128 tokens; a query
that is not reaches dk, and a cotangent dv, of the keys behind it in its tile.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib, _validate
from .varlen import _bounds


def _check(q, k, v, bounds, scale):
    """Bounds and scale as the library takes them, if everything is as it should be."""

    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    for name, x in (("q", q), ("k", k), ("v", v)):
        _validate.heads_tensor(name, x, q.device, q.dtype)
    if k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("k and v must have the same shape, and q's [B, T] and D")
    if min(q.shape[0], q.shape[2], k.shape[2]) <= 0:
        raise ValueError("batch and heads must be positive")
    if q.shape[2] % k.shape[2]:
        raise ValueError("the number of query heads must be a multiple of that of key heads")
    _lib.require_b200(q.device)
    if bounds is not None:
        bounds = _bounds(bounds, q.shape[1])
    return bounds, _validate.float32_scale(scale, q.shape[3])


def _sequences(q, bounds):
    """``(host bounds or None, number of sequences, rows of one or of all)`` as the library takes them."""

    if bounds is None:
        return None, q.shape[0], q.shape[1]
    return _lib.int64s(*bounds), len(bounds) - 1, q.shape[1]


_SHORT = 128     # GDN2_WINDOW_SHORT_ROWS


def _launches(bounds, apart=False) -> int:
    """Launches of a pass: one, or one for every 256 packed sequences of which any has a token; with ``apart`` another one for
    short sequences beside longer ones."""

    if bounds is None:
        return 1
    lengths = [b - a for a, b in zip(bounds, bounds[1:])]
    groups = [lengths[i:i + 256] for i in range(0, len(lengths), 256)]
    if not apart:
        return sum(any(group) for group in groups)
    return sum(len({n > _SHORT for n in group if n > 0}) for group in groups)


def _apart(q, bounds, window) -> bool:
    """Whether a training forward with a window takes short sequences apart: the window reaches over all of them."""

    return window != (0, 0) and window[0] >= (q.shape[1] if bounds is None else max(b - a for a, b in zip(bounds, bounds[1:])))


def _keeps_rest(q, bounds, window) -> bool:
    """Whether a backward with a window reads what the output's rounding has left over: of all sequences, or of short ones."""

    if not _apart(q, bounds, window):
        return window != (0, 0)
    return q.shape[1] <= _SHORT if bounds is None else any(a < b <= a + _SHORT for a, b in zip(bounds, bounds[1:]))


def _entry(name, window):
    """The entry point ``name`` of attention without a window or with one, and what says so."""

    return f"gdn2_{name}" if window == (0, 0) else f"gdn2_window_{name}", () if window == (0, 0) else window


def _forward(q, k, v, bounds, scale, window, training):
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    if q.shape[1] == 0:
        return out, None, None
    host, n_seq, rows = _sequences(q, bounds)
    statistics = None
    if training:
        each = _lib.lib().gdn2_attention_stat_rows(host, n_seq, rows)
        if each < 0:
            _lib.check(int(each), "gdn2_attention_stat_rows")
        statistics = torch.empty((2, q.shape[2], each), device=q.device, dtype=torch.float32)
    strides = _lib.int64s(*(s for x in (q, k, v) for s in _validate.head_strides(x)))
    name, more = _entry("attention_forward", window)
    rest = torch.empty_like(out) if training and _keeps_rest(q, bounds, window) else None    # what the output's rounding leaves over
    _lib.call(name, q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
              _lib.ptr(statistics), *((_lib.ptr(rest),) if more else ()), strides, host, n_seq, rows, q.shape[2], k.shape[2], q.shape[3], *more,
              _lib.dtype_code(q.dtype), scale, _lib.stream_ptr(q.device), kernels=_launches(bounds, rest is not None and _apart(q, bounds, window)))
    return out, statistics, rest


class _CausalAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bounds, scale, window):
        done = _native(q, k, v, bounds, scale, window, True)
        if done is None:
            bounds, scale = _check(q, k, v, bounds, scale)
            done = _forward(*(_validate.detached(x) for x in (q, k, v)), bounds, scale, window, True)
        out, statistics, rest = done
        ctx.save_for_backward(q, k, v, out, statistics, rest)
        ctx.bounds, ctx.scale, ctx.window = bounds, scale, window
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        q, k, v, out, statistics, rest = ctx.saved_tensors
        if statistics is not None and _lib.KERNEL_EVENTS is None:
            done = _lib.host().attention_backward(q, k, v, out, statistics, d_out, ctx.bounds, ctx.scale, *ctx.window, rest)
            if done is not None:
                return (*done, None, None, None)
        scale = _validate.float32_scale(ctx.scale, q.shape[3])
        q, k, v = (_validate.detached(x) for x in (q, k, v))
        grads = tuple(torch.empty(x.shape, device=x.device, dtype=x.dtype) for x in (q, k, v))
        if statistics is None:
            return (*grads, None, None, None)
        if d_out.stride(3) != 1 or d_out.data_ptr() % 16 or any(
                n > 1 and (s <= 0 or s % 8) for n, s in zip(d_out.shape[:3], d_out.stride())):
            d_out = d_out.clone(memory_format=torch.contiguous_format)
        host, n_seq, rows = _sequences(q, ctx.bounds)
        strides = _lib.int64s(*(s for x in (q, k, v, d_out) for s in _validate.head_strides(x)))
        name, more = _entry("attention_backward", ctx.window)
        with torch.cuda.device(q.device):
            size = getattr(_lib.lib(), name + "_bytes")(host, n_seq, rows, q.shape[2], k.shape[2], q.shape[3], *more)
        if size < 0:
            _lib.check(int(size), name + "_bytes")
        scratch = torch.empty(size, device=q.device, dtype=torch.uint8)
        _lib.call(name, q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                  *((_lib.ptr(rest),) if more else ()), d_out.data_ptr(), statistics.data_ptr(), scratch.data_ptr(), *(x.data_ptr() for x in grads), strides,
                  host, n_seq, rows, q.shape[2], k.shape[2], q.shape[3], *more, _lib.dtype_code(q.dtype), scale,
                  _lib.stream_ptr(q.device), kernels=(3 + (size > 2 * statistics.numel() + 15)) * _launches(ctx.bounds))
        return (*grads, None, None, None)


def _native(q, k, v, bounds, scale, window, training):
    """The call on the native host path, ``(output, statistics, rest)``; None where it is not the plain case."""

    if _lib.KERNEL_EVENTS is not None or not getattr(q, "is_cuda", False):
        return None
    return _lib.host().attention_forward(q, k, v, bounds, scale, *window, training)


def _attention(q, k, v, bounds, scale, window=(0, 0)):
    if forward_ad._current_level >= 0:
        _validate.refuse_tangents("causal attention" if window == (0, 0) else "attention with a window", q, k, v)
    if torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad for x in (q, k, v)):
        return _CausalAttention.apply(q, k, v, bounds, scale, window)
    done = _native(q, k, v, bounds, scale, window, False)
    if done is None:
        bounds, scale = _check(q, k, v, bounds, scale)
        done = _forward(*(_validate.detached(x) for x in (q, k, v)), bounds, scale, window, False)
    return done[0]


def _packed_bounds(q, cu_seqlens):
    """Cumulative lengths of packed sequences as a tuple."""

    if not isinstance(q, torch.Tensor) or q.ndim != 4 or q.shape[0] != 1:
        raise ValueError("packed sequence tensors must have shape [1, total, H, D]")
    return cu_seqlens if isinstance(cu_seqlens, tuple) else _bounds(cu_seqlens, q.shape[1])


def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None) -> torch.Tensor:
    """Softmax attention of every token over itself and the tokens before it.

    ``q [B, T, Hq, D]``, ``k`` and ``v [B, T, Hkv, D]``, fp16 or bf16, ``D`` a multiple of 8 up to 128, ``Hq`` a multiple
    of ``Hkv``; views are fine where their rows of channels are 16-byte aligned.  ``scale`` defaults to ``D ** -0.5``.
    Returns a contiguous tensor like ``q``; differentiable in ``q``, ``k`` and ``v``."""

    return _attention(q, k, v, None, scale)


def causal_attention_varlen(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens,
    *,
    scale: float | None = None,
) -> torch.Tensor:
    """``causal_attention`` over ``N`` sequences packed along time.

    Tensors are ``[1, total, H, D]``; ``cu_seqlens`` holds ``N + 1`` cumulative lengths (tensor or sequence of ints, read
    on the host).  No token sees one of another sequence, whatever stands there."""

    return _attention(q, k, v, _packed_bounds(q, cu_seqlens), scale)


__all__ = ["causal_attention", "causal_attention_varlen"]
