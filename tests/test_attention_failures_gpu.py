"""GPU tests of the waits inside the attention kernels: one that runs out ends the CTA by itself and leaves NaN, never a number
that lacks a part of its sum.  ``gdn2_debug_wait_limit(0)`` makes every wait look once, so that those which have anything to
wait for run out at once; nothing hangs or faults, and the next call is as any other."""

from __future__ import annotations

import contextlib

import pytest
import torch

from gdn2_sm120_b200 import _lib
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen
from gdn2_sm120_b200.paged import tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@contextlib.contextmanager
def _no_waiting():
    assert _lib.lib().gdn2_debug_wait_limit(0) == 0
    try:
        yield
    finally:
        assert _lib.lib().gdn2_debug_wait_limit(-1) == 0


def _inputs(lead, heads, kv_heads, dim, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(*lead, h, dim, generator=gen, device=DEV).to(BF16) for h in (heads, kv_heads, kv_heads, heads)]


def _right_or_nan(call, repeats=8):
    want = call()
    for _ in range(repeats):
        with _no_waiting():
            got = call()
            torch.cuda.synchronize()
        for a, b in zip(got, want):
            nan = torch.isnan(a)
            assert nan.any() and torch.equal(a[~nan], b[~nan])
    assert all(torch.equal(a, b) for a, b in zip(call(), want))


@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [((700, 700), 4, 2, 128), ((1000,), 2, 1, 64), ((64,), 1, 1, 64), ((300, 1, 77), 6, 3, 96)])
def test_causal_attention(lengths, heads, kv_heads, dim):
    total = sum(lengths)
    bounds = tuple(sum(lengths[:i]) for i in range(len(lengths) + 1))
    q, k, v, _ = _inputs((1, total), heads, kv_heads, dim)
    _right_or_nan(lambda: [causal_attention_varlen(q, k, v, bounds)])
    _right_or_nan(lambda: [causal_attention(q, k, v)])


@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [((700, 700), 4, 2, 128), ((1000,), 2, 1, 64), ((64,), 1, 1, 64), ((300, 1, 77), 6, 3, 96),
                                                         ((2048,), 8, 1, 128)])
def test_gradients(lengths, heads, kv_heads, dim):
    total = sum(lengths)
    bounds = tuple(sum(lengths[:i]) for i in range(len(lengths) + 1))
    q, k, v, do = _inputs((1, total), heads, kv_heads, dim)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = causal_attention_varlen(*leaves, bounds)
    _right_or_nan(lambda: torch.autograd.grad(out, leaves, do, retain_graph=True))


@pytest.mark.parametrize("drafted,heads,lengths", [(1, 4, (3000, 40)), (4, 8, (100,)), (20, 8, (5000,)), (30, 4, (77, 0)), (60, 16, (9000, 300)),
                                                   (64, 16, (10,))])
def test_trees(drafted, heads, lengths):
    """Up to 16, 128 and 256 rows of a key head and more, in one CTA's part and shared by several."""

    kv_heads, dim, page, batch = 2, 128, 16, len(lengths)
    q, k, v, _ = _inputs((batch, drafted), heads, kv_heads, dim)
    columns = max(-(-n // page) for n in lengths)
    pages = [torch.randn(batch * columns, page, kv_heads, dim, device=DEV).to(BF16) for _ in range(2)]
    table = torch.arange(batch * columns, device=DEV, dtype=torch.int32).view(batch, columns)
    counts = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    _right_or_nan(lambda: [tree_attention(q, k, v, *pages, table, counts)])


def test_limits_of_the_limit():
    assert _lib.lib().gdn2_debug_wait_limit(2 ** 20) == 0 and _lib.lib().gdn2_debug_wait_limit(2 ** 20 + 1) == -9
    assert _lib.lib().gdn2_debug_wait_limit(-1) == 0
