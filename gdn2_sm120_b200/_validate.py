"""Host-side argument checks shared by the token, chunk and backward wrappers.

The exception types and the key phrases of the messages follow the reference
(src/gdn2_sm120/recurrent.py:374-433, 451-478; chunk.py:1183-1229, 1265-1316;
backward.py:953-1009) because its tests match on them: everything is rejected in
Python, before any launch, and nothing falls back silently.
"""

from __future__ import annotations

import math
import struct

import torch
from torch.autograd import forward_ad

from . import _lib

DIM = 128
_SEQ_NAMES = ("q", "k", "v", "g", "beta", "w")
_LOW_PRECISION = (torch.float16, torch.bfloat16)


def sequence_inputs(q, k, v, g, beta, w, *, dim_error=ValueError, need_tokens=False,
                    need_alignment=False):
    """Validate the six ``[B, T, H, 128]`` tensors; return ``(B, T, H)``."""

    seq = (q, k, v, g, beta, w)
    if not all(isinstance(x, torch.Tensor) for x in seq):
        raise TypeError("q, k, v, g, beta, and w must be torch.Tensor objects")
    if any(x.ndim != 4 for x in seq):
        raise ValueError("q, k, v, g, beta, and w must be rank-4 [B, T, H, D] tensors")
    if not (q.shape == k.shape == g.shape == beta.shape):
        raise ValueError("q, k, g, and beta must have identical [B, T, H, K] shapes")
    if v.shape != w.shape or v.shape[:3] != q.shape[:3]:
        raise ValueError("v and w must match each other and q's [B, T, H] dimensions")
    batch, time, heads, key_dim = q.shape
    if key_dim != DIM or v.shape[-1] != DIM:
        raise dim_error("the B200 GDN2 kernels require K == V == 128")
    if batch <= 0 or heads <= 0 or (need_tokens and time <= 0):
        what = "batch, time, and heads" if need_tokens else "batch and heads"
        raise ValueError(f"{what} must be positive")
    if q.dtype not in _LOW_PRECISION:
        raise TypeError("q/k/v/beta/w must use torch.float16 or torch.bfloat16")
    if any(x.dtype != q.dtype for x in (k, v, beta, w)):
        raise TypeError("q, k, v, beta, and w must have the same dtype")
    if g.dtype not in (q.dtype, torch.float32):
        raise TypeError("g must have the input dtype or torch.float32")
    if not all(x.is_cuda for x in seq):
        raise ValueError("all inputs must be CUDA tensors")
    if any(x.device != q.device for x in seq):
        raise ValueError("all inputs must be on the same CUDA device")
    if not all(x.is_contiguous() for x in seq):
        raise ValueError("all inputs must be contiguous")
    if need_alignment and any(x.data_ptr() % 16 for x in seq):
        raise ValueError("all inputs must be 16-byte aligned")
    _lib.require_b200(q.device)
    return batch, time, heads


def state(name: str, tensor, batch: int, heads: int, device, *, need_alignment=False):
    """Validate an fp32 ``[B, H, 128, 128]`` state tensor."""

    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor or None")
    expected = (batch, heads, DIM, DIM)
    if tuple(tensor.shape) != expected:
        raise ValueError(f"{name} must have shape {expected}")
    if tensor.dtype != torch.float32:
        raise TypeError(f"{name} must use torch.float32")
    if tensor.device != device:
        raise ValueError(f"{name} must be on the same CUDA device as q")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if need_alignment and tensor.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")


def buffer(name: str, tensor, shape, dtype, device, *, need_alignment=False):
    """Validate a caller-provided output buffer."""

    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor or None")
    if tuple(tensor.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}")
    if tensor.dtype != dtype:
        raise TypeError(f"{name} must use {dtype}")
    if tensor.device != device:
        raise ValueError(f"{name} must be on the same CUDA device as q")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if need_alignment and tensor.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned for the chunk path")


def float32_scale(scale, dim: int = DIM) -> float:
    """Default 1/sqrt(dim); reject values that are not finite once rounded to fp32."""

    value = float(scale) if scale is not None else 1.0 / math.sqrt(dim)
    if not math.isfinite(value):
        raise ValueError("scale must be finite")
    try:
        rounded = struct.unpack("=f", struct.pack("=f", value))[0]
    except OverflowError as exc:
        raise ValueError("scale must be representable as float32") from exc
    if not math.isfinite(rounded):
        raise ValueError("scale must be representable as float32 (finite after rounding)")
    return rounded


def byte_span(tensor: torch.Tensor) -> tuple[int, int]:
    """Half-open byte interval of a contiguous tensor."""

    lo = tensor.data_ptr()
    return lo, lo + tensor.numel() * tensor.element_size()


def extent(tensor: torch.Tensor) -> tuple[int, int]:
    """Half-open byte interval from the first to the last element of a strided tensor."""

    lo = tensor.data_ptr()
    if tensor.numel() == 0:
        return lo, lo
    return lo, lo + (sum((n - 1) * s for n, s in zip(tensor.shape, tensor.stride())) + 1) * tensor.element_size()


def heads_tensor(name: str, tensor, device, dtype) -> None:
    """Validate one ``[B, T, H, D]`` operand of attention: a view is fine where every row of channels is 16-byte
    aligned (the kernels' tiled copies need that) and no two elements share a place."""

    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tensor.ndim != 4:
        raise ValueError(f"{name} must be a rank-4 [B, T, H, D] tensor")
    if dtype not in _LOW_PRECISION:
        raise TypeError("attention takes torch.float16 or torch.bfloat16")
    if tensor.dtype != dtype:
        raise TypeError(f"{name} must have q's dtype")
    if not tensor.is_cuda or tensor.device != device:
        raise ValueError("all inputs must be CUDA tensors on the same device")
    dim = tensor.shape[3]
    if not 0 < dim <= 128 or dim % 8:
        raise NotImplementedError("attention takes head dimensions that are multiples of 8, up to 128")
    if tensor.stride(3) != 1:
        raise ValueError(f"the channels of {name} must be contiguous")
    if tensor.data_ptr() % 16 or any(n > 1 and (s <= 0 or s % 8) for n, s in zip(tensor.shape[:3], tensor.stride())):
        raise ValueError(f"every row of {name} must be 16-byte aligned and have a place of its own")


def head_strides(tensor: torch.Tensor) -> tuple[int, int, int]:
    """Batch, token and head stride in elements; a dimension of size 1 gets that of a contiguous tensor."""

    _, time, heads, dim = tensor.shape
    dense = (time * heads * dim, heads * dim, dim)
    return tuple(d if n <= 1 else s for n, s, d in zip(tensor.shape, tensor.stride(), dense))


def spans_overlap(left: tuple[int, int], right: tuple[int, int]) -> bool:
    """True when two non-empty half-open intervals intersect."""

    if left[0] >= left[1] or right[0] >= right[1]:
        return False
    return left[0] < right[1] and right[0] < left[1]


def _sums_to(terms, target, tries=20000):
    """Whether ``target`` is a sum of ``stride * y`` with ``lo <= y <= hi`` for ``(stride, lo, hi)`` in ``terms``.  Largest
    strides first, every choice bounded by what the smaller ones can still make up for: a try or two a stride in layouts
    that nest.  True where that many tries do not tell."""

    terms.sort(reverse=True)
    reach = [(0, 0)]                        # least and most of the terms behind
    for stride, lo, hi in terms[:0:-1]:
        reach.append((reach[-1][0] + stride * lo, reach[-1][1] + stride * hi))
    reach.reverse()
    open_ends = [(0, target)]
    while open_ends:
        i, target = open_ends.pop()
        if i == len(terms):
            if target == 0:
                return True
            continue
        (stride, lo, hi), (least, most) = terms[i], reach[i]
        for y in range(max(lo, -((most - target) // stride)), min(hi, (target - least) // stride) + 1):
            open_ends.append((i + 1, target - stride * y))
            tries -= 1
        if tries < 0:
            return True
    return False


def _places(tensor: torch.Tensor):
    """First byte, byte behind the last, and ``(bytes, size)`` of the dimensions that have more than one place."""

    size = tensor.element_size()
    lo, dims = tensor.data_ptr(), [(s * size, n) for s, n in zip(tensor.stride(), tensor.shape) if n != 1]
    return lo, lo + sum((n - 1) * s for s, n in dims) + size if tensor.numel() else lo, dims


def share_elements(left: torch.Tensor, right: torch.Tensor) -> bool:
    """True when two strided tensors have a byte in common (slices of one projection have none, though their extents meet)."""

    lo, end, dims = _places(left)
    other_lo, other_end, other_dims = _places(right)
    if not spans_overlap((lo, end), (other_lo, other_end)):
        return False
    ranges = {1: [1 - right.element_size(), left.element_size() - 1]}
    for s, n in dims:
        if s:
            ranges.setdefault(s, [0, 0])[1] += n - 1
    for s, n in other_dims:
        if s:
            ranges.setdefault(s, [0, 0])[0] -= n - 1
    return _sums_to([(s, lo, hi) for s, (lo, hi) in ranges.items()], other_lo - lo)


def shares_with_itself(tensor: torch.Tensor) -> bool:
    """True when two elements of a strided tensor share a place."""

    if tensor.is_contiguous() or tensor.numel() == 0:
        return False
    dims = sorted(_places(tensor)[2])
    behind, nests = tensor.element_size(), True
    for s, n in dims:
        nests = nests and s >= behind       # every stride passes all that the smaller ones reach
        behind += (n - 1) * s
    if nests:
        return False
    reach = 0
    for i, (s, n) in enumerate(dims):       # the largest stride in which two places differ
        if s == 0 or any(_sums_to([(t, 1 - m, m - 1) for t, m in dims[:i]], s * y) for y in range(1, min(n - 1, reach // s) + 1)):
            return True
        reach += (n - 1) * s
    return False


def heads_in_place(q: torch.Tensor, k: torch.Tensor, read) -> None:
    """Raise where two ``[B, T, H, D]`` tensors of one type, which a call writes to, share elements, or overlap what it reads
    (contiguous tensors)."""

    size, a, b = q.element_size(), q.data_ptr(), k.data_ptr()
    q_stride, k_stride = q.stride(), k.stride()
    batch, time, heads, dim = q.shape
    first, second = (heads, k.shape[2]) if a <= b else (k.shape[2], heads)
    span = abs(a - b) // size + second * dim
    reach = span + (time - 1) * q_stride[1]
    if (q_stride[2:] == (dim, 1) == k_stride[2:] and span >= (first + second) * dim
            and (time == 1 or span <= q_stride[1] == k_stride[1]) and (batch == 1 or reach <= q_stride[0] == k_stride[0])):
        # slices of one projection: a token's heads of both lie behind one another, then comes the next token
        spans = [(min(a, b), min(a, b) + (reach + (batch - 1) * q_stride[0]) * size)]
    else:
        spans = [byte_span(x) if x.is_contiguous() else extent(x) for x in (q, k)]
        if shares_with_itself(q) or shares_with_itself(k) or (spans_overlap(*spans) and share_elements(q, k)):
            raise ValueError("inplace=True needs tensors whose elements have places of their own")
    for x in read:
        if x is not None:
            lo, end = byte_span(x)
            for from_, to in spans:
                if lo < to and from_ < end:
                    raise ValueError("inplace=True needs cos, sin, and positions that do not lie in q or k")


def refuse_tangents(what: str, *tensors) -> None:
    """Raise where a tensor is a dual one of forward-mode differentiation, whose tangent the kernels would drop.  To be called
    where ``forward_ad._current_level`` is not negative: asking for that costs a small call nothing."""

    if any(isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative: call it with the primal tensors")


def detached(tensor):
    """Storage-sharing view without an autograd edge (``None`` passes through)."""

    if tensor is None or not tensor.requires_grad:
        return tensor
    return tensor.detach()
