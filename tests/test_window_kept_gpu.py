"""GPU tests of what a training forward with a window keeps for its backward: nothing that is not read there."""

from __future__ import annotations

import gc

import pytest
import torch

from gdn2_sm120_b200 import _lib
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen
from gdn2_sm120_b200.window import window_attention, window_attention_varlen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _inputs(lead, heads, kv_heads, dim, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(*lead, h, dim, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads, kv_heads, heads)]


def _bounds(lengths):
    return tuple(sum(lengths[:i]) for i in range(len(lengths) + 1))


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("lengths", [(300, 300), (129, 700)])
def test_nothing_is_kept_that_the_backward_does_not_read(lengths, python):
    bounds = _bounds(lengths)
    q, k, v, _ = _inputs((1, bounds[-1]), 4, 2, 64, BF16, seed=8)
    q.requires_grad_(True)
    gc.collect()      # what earlier tests have left does not go away meanwhile

    def held(call, *args):
        before = torch.cuda.memory_allocated()
        out = call(q, k, v, *args)
        return torch.cuda.memory_allocated() - before, out

    _lib.KERNEL_EVENTS = {} if python else None
    try:
        want = held(causal_attention_varlen, bounds)[0]
        assert held(window_attention_varlen, bounds, 700)[0] == want
        assert held(window_attention_varlen, bounds, 100)[0] > want     # (its delta is taken from what rounding left over, too)
        if len(set(lengths)) == 1:
            x = [y.view(2, 300, -1, 64) for y in (q, k, v)]
            before = torch.cuda.memory_allocated()
            out = window_attention(*x, 300)
            used = torch.cuda.memory_allocated() - before
            del out
            before = torch.cuda.memory_allocated()
            out = causal_attention(*x)
            assert torch.cuda.memory_allocated() - before == used
    finally:
        _lib.KERNEL_EVENTS = None
