"""GPU tests of gradients where a window reaches over whole sequences: a short one's do not depend on what it is packed with."""

from __future__ import annotations

import math

import pytest
import torch

from gdn2_sm120_b200 import _lib
from gdn2_sm120_b200.attention import causal_attention_varlen
from gdn2_sm120_b200.window import window_attention, window_attention_varlen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(lead, heads, kv_heads, dim, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(*lead, h, dim, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads, kv_heads, heads)]


def _run(call, q, k, v, do, *args, **more):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = call(*leaves, *args, **more)
    return out.detach(), *torch.autograd.grad(out, leaves, do)


def _bounds(lengths):
    return tuple(sum(lengths[:i]) for i in range(len(lengths) + 1))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("time,others", [(3, (129,)), (11, (300, 0, 1000)), (100, (129,)), (3, (128,)), (11, ())])
def test_gradients_of_short_sequences_beside_longer_ones(dtype, time, others):
    # the bound on dq and dk is that of test_gradients_of_few_keys_are_off_by_two_roundings, where it is derived
    heads, dim, count = 8, 64, max(1, 2400 // time)
    bounds = _bounds((time,) * (count // 2) + others + (time,) * (count - count // 2))
    short = torch.ones(bounds[-1], device=DEV, dtype=torch.bool)
    short[time * (count // 2):bounds[-1] - time * (count - count // 2)] = False
    q, k, v, do = _inputs((1, bounds[-1]), heads, heads, dim, dtype, seed=5)
    got = _run(window_attention_varlen, q, k, v, do, bounds, 2000)
    leaves = [x[0, short].view(count, time, heads, dim).double().transpose(1, 2).requires_grad_(True) for x in (q, k, v)]
    scores = (leaves[0] @ leaves[1].transpose(-1, -2) * dim ** -0.5).masked_fill(~torch.ones(time, time, device=DEV, dtype=torch.bool).tril(), -math.inf)
    cotangent = do[0, short].view(count, time, heads, dim).double().transpose(1, 2)
    want = torch.autograd.grad(scores.softmax(-1) @ leaves[2], leaves, cotangent)
    for name, x, y in zip(("dq", "dk"), got[1:3], want):
        y = y.transpose(1, 2)
        rounding = (y.to(dtype).double() - y).norm()
        assert (x[0, short].view(y.shape).double() - y).norm() < 1.65 * rounding, name


@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [
    ((3, 129), 2, 1, 64), ((128, 129, 1, 0, 700, 64), 4, 2, 128), ((1,) * 300 + (500,) * 3 + (90,) * 5, 4, 4, 40), ((2000, 5), 16, 1, 128), ((400,) * 3 + (2,) * 253, 2, 1, 64),
    ((2,) * 256 + (400,) * 3, 2, 1, 64),
])
def test_a_sequence_alone_and_beside_others(lengths, heads, kv_heads, dim):
    """Bit for bit, and longer sequences as in causal attention."""

    bounds = _bounds(lengths)
    q, k, v, do = _inputs((1, bounds[-1]), heads, kv_heads, dim, BF16, seed=6)
    got = _run(window_attention_varlen, q, k, v, do, bounds, 3000, sinks=2)
    causal = _run(causal_attention_varlen, q, k, v, do, bounds)
    assert torch.equal(got[0], causal[0])
    assert torch.equal(got[0], window_attention_varlen(q, k, v, bounds, 3000, sinks=2))
    for i in {0, 1, 2, len(lengths) // 2, len(lengths) - 3, len(lengths) - 2, len(lengths) - 1} & set(range(len(lengths))):
        part = slice(bounds[i], bounds[i + 1])
        if lengths[i] > 128:
            assert all(torch.equal(a[:, part], b[:, part]) for a, b in zip(got, causal))
        elif lengths[i] > 0:
            alone = _run(window_attention, *(x[:, part] for x in (q, k, v, do)), lengths[i])
            # (a key's gradients may be sums of parts, as many as the whole call has, in 32 bits)
            assert torch.equal(got[0][:, part], alone[0]) and torch.equal(got[1][:, part], alone[1])
            for a, b in zip(got[2:], alone[2:]):
                assert torch.equal(a[:, part], b) or (heads // kv_heads >= 16 and (a[:, part] - b).abs().max() <= 2.0 ** -7 * b.abs().max())
    assert all(torch.equal(a, b) for a, b in zip(got, _run(window_attention_varlen, q, k, v, do, bounds, 3000, sinks=2)))


def test_both_host_paths_and_their_launches():
    bounds = _bounds((3, 300, 1, 200) + (0,) * 300 + (50, 129) + (7,) * 260)
    inputs = _inputs((1, bounds[-1]), 4, 2, 64, BF16, seed=7)
    results, launches = [], []
    for events in (None, {}):
        _lib.LAUNCHES[0] = 0
        _lib.KERNEL_EVENTS = events       # calls that are timed one by one go through Python
        try:
            results.append(_run(window_attention_varlen, *inputs, bounds, 300))
        finally:
            _lib.KERNEL_EVENTS = None
        launches.append(_lib.LAUNCHES[0])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    # 566 sequences: short and long ones among the first 256 and the next, short ones among the last 54, for each of which the
    # backward has delta, keys and queries
    assert launches == [2 + 2 + 1 + 3 * 3] * 2
