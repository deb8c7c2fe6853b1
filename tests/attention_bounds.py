"""Plain attention in 64 bits with elementwise bounds on what kernels may be off, for the attention tests.

With u the unit roundoff of the tensors' type, a kernel that keeps scores, weights, statistics and sums in 32 bits rounds

  a weight once, for its product with the values:   |o' - o| <= u sum_j p_ij |v_j| =: u A_i
  the output once:                                  + u |o|
  in the backward, p and ds once each:              dv: u sum_i p_ij |do_i|;  dq, dk: u sum |ds| |k| and u sum |ds| |q|
  and takes delta_i = do_i . o_i from that output:  |delta' - delta| <= u sum_c |do_c| (|o_c| + A_c) =: E_i, so ds is off
                                                    by p_ij E_i more
  a gradient once:                                  + u |gradient|

and floats below their normal range have a fixed spacing, half of which a value may be off, or count as 0.  Everything in 32 bits
(exponentials to 2^-21, sums of some hundred terms, scores of some tens) adds less than 2^-13 of the same sums of magnitudes;
`SLACK` covers that and the products of two roundings."""

from __future__ import annotations

import math

import torch

SLACK = 1.05
FP32 = 2.0 ** -13


def unit(dtype) -> float:
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11   # 8 and 11 significant bits, half a unit in the last


def spacing(dtype) -> float:
    """Half the distance of neighbours below the normal range, or where that is the 32-bit floats' own (bf16) its end:
    what is smaller counts as 0."""

    return 2.0 ** -126 if dtype == torch.bfloat16 else 2.0 ** -25


def attention(q, k, v, seen, scale, do=None):
    """``q [H, N, D]``, ``k`` and ``v [Hkv, M, D]``, ``seen [N, M]``: ``{name: (value, bound)}`` of o, dq, dk, dv.
    Masked places of k and v may hold anything.  Rows that see nothing give 0."""

    dtype = q.dtype
    u, tiny = unit(dtype), spacing(dtype)
    group = q.shape[0] // k.shape[0]
    q, k, v = q.double(), k.double(), v.double()
    kk, vv = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    s = (q @ kk.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    o, a = p @ vv, p @ vv.abs()
    spread = seen.double() @ vv.abs() * tiny          # weights in the subnormal range; the largest one is 1 or more
    bounds = {"o": (o, SLACK * u * (o.abs() + a) + FP32 * a + spread + tiny)}
    if do is None:
        return bounds
    do = do.double()
    dp = do @ vv.transpose(1, 2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    off = u * (do.abs() * (o.abs() + a + spread / u)).sum(-1, keepdim=True)
    size = p * (do.abs() @ vv.abs().transpose(1, 2) + delta.abs())   # what 32-bit sums of dp and ds are off by
    ds_off = SLACK * (u * ds.abs() + p * off) + FP32 * size + tiny * seen

    def shared(x):
        return x.view(k.shape[0], group, *x.shape[1:]).sum(1)

    def grad(value, error):
        return value, SLACK * (u * value.abs() + error) + tiny

    c = abs(scale)
    bounds["dq"] = grad(scale * ds @ kk, c * ds_off @ kk.abs())
    bounds["dk"] = grad(shared(scale * ds.transpose(1, 2) @ q), shared(c * ds_off.transpose(1, 2) @ q.abs()))
    bounds["dv"] = grad(shared(p.transpose(1, 2) @ do),
                        shared(((u + FP32) * p + tiny * seen).transpose(1, 2) @ do.abs()))
    return bounds


def causal(rows, device):
    return torch.ones(rows, rows, dtype=torch.bool, device=device).tril()


def check(name, got, value, bound):
    """`got` [N, H, D] against value and bound [H, N, D]."""

    error = (got.double().transpose(0, 1) - value).abs()
    worst = (error / bound.clamp_min(1e-300)).max().item() if error.numel() else 0.0
    assert torch.isfinite(got).all(), f"{name}: not finite"
    assert worst <= 1.0, f"{name}: {worst:.3f} times its bound"
