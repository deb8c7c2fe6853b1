"""GPU tests of attention with a window over sequences whose values are not all finite: many such items of a CTA in a row, of one
tile of queries and of two."""

from __future__ import annotations

import contextlib
import math

import pytest
import torch

from gdn2_sm120_b200 import _lib
from gdn2_sm120_b200.window import window_attention, window_attention_varlen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


@contextlib.contextmanager
def _short_waits():
    """A wait for what does not come ends after a quarter of a second at most, and leaves NaN."""

    assert _lib.lib().gdn2_debug_wait_limit(1 << 16) == 0
    try:
        yield
    finally:
        assert _lib.lib().gdn2_debug_wait_limit(-1) == 0


def _seen(time, window, sinks):
    i, j = torch.arange(time, device=DEV)[:, None], torch.arange(time, device=DEV)
    return (j <= i) & ((i - j < window) | (j < sinks))


@pytest.mark.parametrize("training", [False, True])
@pytest.mark.parametrize("lengths,window,sinks,heads,kv_heads,dim,dtype", [
    ([100] * 64, 20, 0, 16, 4, 64, BF16), ([100] * 64, 99, 3, 16, 4, 128, FP16), ([60] * 64, 300, 0, 16, 4, 64, BF16), ([1] * 128, 1, 0, 16, 2, 64, BF16),
    ([1 + 37 * i % 128 for i in range(128)], 20, 4, 8, 4, 128, BF16), ([257 + 31 * i % 128 for i in range(40)], 70, 0, 16, 4, 64, FP16),
    ([(1 + 53 * i % 128) + 256 * (i % 3) for i in range(60)], 130, 5, 12, 4, 128, BF16), ([1 + 71 * i % 500 for i in range(60)], 33, 130, 12, 4, 64, BF16),
])
def test_values_that_are_not_finite_in_many_sequences(lengths, window, sinks, heads, kv_heads, dim, dtype, training):
    bounds = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    gen = torch.Generator(device=DEV).manual_seed(sum(lengths))
    q, k, v = (torch.randn(1, bounds[-1], h, dim, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads, kv_heads))
    group, even = heads // kv_heads, len(set(lengths)) == 1

    def run(v):
        x = [y.detach().requires_grad_(training) for y in (q, k, v)]
        with _short_waits():
            outs = [window_attention_varlen(*x, bounds, window, sinks=sinks)]
            if even:
                outs.append(window_attention(*(y.view(len(lengths), lengths[0], -1, dim) for y in x), window, sinks=sinks).view(q.shape))
            torch.cuda.synchronize()
        return [y.detach() for y in outs]

    clean = run(v)
    assert all(torch.isfinite(x).all() for x in clean)
    for stride in (1, 2, 3):          # every sequence, every second one, ...
        strange, reached = v.clone(), torch.zeros_like(q, dtype=torch.bool)
        for b in range(0, len(lengths), stride):
            part = slice(bounds[b], bounds[b + 1])
            seen = _seen(lengths[b], window, sinks)
            for row in {b % lengths[b], lengths[b] // 2, lengths[b] - 1}:
                head, channel = (b + row) % kv_heads, (7 * row + b) % dim
                strange[0, bounds[b] + row, head, channel] = (math.nan, math.inf, -math.inf)[(row + b) % 3]
                reached[0, part, head * group:(head + 1) * group, channel] |= seen[:, row, None]
        for got, want in zip(run(strange), clean):
            assert torch.equal(got[~reached], want[~reached]) and not torch.isfinite(got[reached]).any()
