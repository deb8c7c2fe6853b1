"""Rotary positions for the attention layers that stand between Gated DeltaNet-2 layers.

``rotary_tables``   cosines and sines of the angles, for plain and for stretched contexts
``apply_rotary``    turns queries and keys by them in one launch (csrc/rotary.cu), with its gradient

Channel pair ``i`` of a head turns by ``position * base ** (-2 i / rotated)``.  A pair is ``(i, i + rotated / 2)`` in the
``"half"`` layout and ``(2 i, 2 i + 1)`` in the ``"interleaved"`` one; channels from ``rotated`` on are left as they are.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib, _validate

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_LAYOUTS = ("half", "interleaved")
_SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_tables(
    positions: int,
    rotated: int,
    *,
    base: float = 10000.0,
    scaling: str | None = None,
    factor: float = 1.0,
    trained: int | None = None,
    fast: float = 32.0,
    slow: float = 1.0,
    device="cuda",
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(cos, sin)``, fp32 ``[positions, rotated / 2]``, from angles in 64 bits (at position 10 ** 6 an angle in 32 bits
    is off by 0.06).

    ``scaling`` serves contexts ``factor`` times as long as a model was trained on:

    ``"linear"``  positions are divided by ``factor``
    ``"ntk"``     the base grows to ``base * factor ** (rotated / (rotated - 2))``: the slowest pair turns ``factor``
                  times as slowly, the fastest as before
    ``"yarn"``    a pair that turns ``r`` times in ``trained`` positions keeps its speed from ``r = fast`` on, is slowed
                  ``factor`` times up to ``r = slow``, and lies linearly between the two in between; cosines and sines
                  are multiplied by ``1 + 0.1 ln(factor)``, which sharpens the softmax.  Linearly in ``r``, that is, as the
                  method is defined; there are models whose tables are linear in the pair's number ``i`` between the pairs
                  that turn ``fast`` and ``slow`` times.  Both agree at the ends but not in between (128 channels, base 10000,
                  4096 positions, factor 8: pair 33 turns 0.46 times as fast here as there), so a model needs the tables that
                  it was trained with
    """

    if isinstance(positions, bool) or not isinstance(positions, int) or positions <= 0:
        raise ValueError("positions must be a positive int")
    if isinstance(rotated, bool) or not isinstance(rotated, int) or rotated <= 0 or rotated % 2:
        raise ValueError("rotated must be a positive even int")
    if scaling not in _SCALINGS:
        raise ValueError(f"scaling must be one of {_SCALINGS}")
    if not (math.isfinite(base) and base > 0.0):
        raise ValueError("base must be positive and finite")
    if not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError("factor must be finite and at least 1")
    amplitude = 1.0
    if scaling == "ntk":
        if rotated == 2:
            raise ValueError("scaling='ntk' needs more than one pair")
        base = base * factor ** (rotated / (rotated - 2))
    pairs = rotated // 2
    speed = base ** (-torch.arange(pairs, dtype=torch.float64, device=device) / pairs)
    if scaling == "linear":
        speed = speed / factor
    elif scaling == "yarn":
        if isinstance(trained, bool) or not isinstance(trained, int) or trained <= 0:
            raise ValueError("scaling='yarn' needs trained, the positive number of positions of the training")
        if not 0.0 < slow < fast < math.inf:
            raise ValueError("fast must be greater than slow, and both positive and finite")
        turns = speed * (trained / (2.0 * math.pi))
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        speed = speed * keep + speed / factor * (1.0 - keep)
        amplitude = 1.0 + 0.1 * math.log(factor)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * speed
    return (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()


def _check(q, k, cos, sin, positions, layout):
    if not all(isinstance(x, torch.Tensor) for x in (q, k, cos, sin)):
        raise TypeError("q, k, cos, and sin must be torch.Tensor objects")
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError("q and k must be rank-4 [B, T, H, D] tensors")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("q and k must have the same [B, T] and D")
    if min(q.shape[0], q.shape[2], k.shape[2]) <= 0:
        raise ValueError("batch and heads must be positive")
    if not 0 < q.shape[3] <= 512 or q.shape[3] % 2:
        raise ValueError("D must be even and at most 512")
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise TypeError("q and k must both use torch.bfloat16, torch.float16 or torch.float32")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be one of {_LAYOUTS}")
    if not all(x.is_cuda and x.device == q.device for x in (q, k, cos, sin)):
        raise ValueError("all inputs must be CUDA tensors on the same device")
    if cos.ndim != 2 or cos.shape != sin.shape or 0 in cos.shape:
        raise ValueError("cos and sin must have the same shape [positions, rotated / 2]")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must use torch.float32")
    if not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous")
    if 2 * cos.shape[1] > q.shape[3]:
        raise ValueError("cos and sin are for more channels than D")
    if q.stride(3) != 1 or k.stride(3) != 1:
        raise ValueError("the channels of q and k must be contiguous")
    if positions is None:
        if q.shape[1] > cos.shape[0]:
            raise ValueError("cos and sin have fewer positions than q and k have tokens")
    else:
        if not isinstance(positions, torch.Tensor):
            raise TypeError("positions must be a torch.Tensor or None")
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must use torch.int32 or torch.int64")
        if positions.device != q.device:
            raise ValueError("positions must be on the same CUDA device as q")
        if positions.shape not in (q.shape[:2], q.shape[1:2]):
            raise ValueError("positions must have shape [B, T] or [T]")
    _lib.require_b200(q.device)
    return None if positions is None else positions.to(torch.int64).contiguous()


def _native(q, k, cos, sin, positions, layout, inverse):
    """The call on the native host path; None where it is not the plain case."""

    if _lib.KERNEL_EVENTS is not None or layout not in _LAYOUTS or not getattr(q, "is_cuda", False):
        return None
    return _lib.host().rotary(q, k, cos, sin, positions, layout == "interleaved", inverse)


def _launch(q, k, q_out, k_out, cos, sin, positions, layout, inverse):
    batch, time, heads, dim = q.shape
    if time == 0:
        return
    strides = _lib.int64s(*(s for x in (q, k, q_out, k_out) for s in x.stride()[:3]))
    _lib.call("gdn2_rotary", q.device, q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), cos.data_ptr(),
              sin.data_ptr(), _lib.ptr(positions), strides,
              0 if positions is None or positions.ndim == 1 else positions.stride(0), batch, time, heads, k.shape[2], dim,
              cos.shape[1], cos.shape[0], int(layout == "interleaved"), int(inverse), _lib.dtype_code(q.dtype),
              _lib.stream_ptr(q.device))


def _contiguous_like(x):
    return torch.empty(x.shape, device=x.device, dtype=x.dtype)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, layout):
        done = _native(q, k, cos, sin, positions, layout, False)
        if done is None:
            positions = _check(q, k, cos, sin, positions, layout)
            done = _contiguous_like(q), _contiguous_like(k)
            _launch(q.detach(), k.detach(), *done, cos, sin, positions, layout, False)
        ctx.save_for_backward(cos, sin, positions)
        ctx.layout = layout
        return done

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        cos, sin, positions = ctx.saved_tensors
        done = _native(dq, dk, cos, sin, positions, ctx.layout, True)
        if done is not None:
            return (*done, None, None, None, None)
        dq, dk = (x if x.stride(3) == 1 else x.contiguous() for x in (dq, dk))
        q_out, k_out = _contiguous_like(dq), _contiguous_like(dk)
        _launch(dq, dk, q_out, k_out, cos, sin, positions, ctx.layout, True)
        return q_out, k_out, None, None, None, None


def apply_rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor | None = None,
    *,
    layout: str = "half",
    inplace: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Turn ``q [B, T, Hq, D]`` and ``k [B, T, Hk, D]`` by the angles of their positions; returns ``(q, k)``.

    bf16, fp16 or fp32, arithmetic in 32 bits; the inputs may be views (slices of one projection) whose channels are
    contiguous.  ``cos`` and ``sin`` are those of ``rotary_tables``, twice their second size channels turn.
    ``positions`` (int32 or int64, ``[B, T]`` or ``[T]``) defaults to a token's number in its sequence; packed and
    continued sequences give theirs.  A position outside the tables makes the token's rotated channels NaN.
    Differentiable in ``q`` and ``k``; ``inplace=True`` turns the tensors themselves (no gradient) and returns them: slices of
    one projection are fine, tensors that share an element are refused."""

    if forward_ad._current_level >= 0:
        _validate.refuse_tangents("apply_rotary", q, k, cos, sin)
    wants_grad = torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad for x in (q, k))
    if not inplace:
        if wants_grad:
            return _Rotary.apply(q, k, cos, sin, positions, layout)
        done = _native(q, k, cos, sin, positions, layout, False)
        if done is not None:
            return done
    positions = _check(q, k, cos, sin, positions, layout)
    if wants_grad:
        raise ValueError("inplace=True has no gradient")
    given = q, k
    q, k = q.detach(), k.detach()
    if inplace:
        _validate.heads_in_place(q, k, (cos, sin, positions))
        q_out, k_out = q, k
    else:
        q_out, k_out = _contiguous_like(q), _contiguous_like(k)
    _launch(q, k, q_out, k_out, cos, sin, positions, layout, False)
    if not inplace:
        return q_out, k_out
    torch.autograd.graph.increment_version(given)     # a backward that has saved them must not use them any more
    return given


__all__ = ["apply_rotary", "rotary_tables"]
