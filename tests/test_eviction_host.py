"""Host-side checks of accumulated weights and eviction that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gdn2_sm120_b200 import _lib
from gdn2_sm120_b200.eviction import evict_tokens, weighed_attention, weighed_attention_varlen, weighed_token_attention
from gdn2_sm120_b200.window import window_tree_attention

Q, K = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
PAGES, WEIGHTS = torch.zeros(4, 16, 1, 64, dtype=torch.bfloat16), torch.zeros(4, 1, 16)
TABLE, LENGTHS = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)


def test_tensors_on_the_cpu_are_refused():
    for call in (lambda: weighed_attention(Q, K, K), lambda: weighed_attention_varlen(Q, K, K, (0, 1)),
                 lambda: weighed_token_attention(Q, K, K, PAGES, PAGES.clone(), WEIGHTS, TABLE, LENGTHS, torch.zeros(1, 1, dtype=torch.int64)),
                 lambda: window_tree_attention(Q, K, K, PAGES, PAGES.clone(), TABLE, LENGTHS, 4),
                 lambda: evict_tokens(PAGES, PAGES.clone(), WEIGHTS, TABLE, LENGTHS, TABLE, 16)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("keep,sinks,recent,error", [
    (0, 0, 0, ValueError), (-1, 0, 0, ValueError), (8, 5, 4, ValueError), (8, -1, 0, ValueError), (8, 0, -1, ValueError), (8.0, 0, 0, TypeError),
    (True, 0, 0, TypeError), (None, 0, 0, TypeError), (8, 1.0, 0, TypeError), (8, 0, "1", TypeError),
])
def test_budgets_that_are_none(keep, sinks, recent, error):
    with pytest.raises(error):
        evict_tokens(PAGES, PAGES, WEIGHTS, TABLE, LENGTHS, TABLE, keep, sinks=sinks, recent=recent)


def test_entry_points_reject_bad_arguments_without_a_gpu():
    handle, one, null = _lib.lib(), ctypes.c_void_p(256), None
    strides = _lib.int64s(*[64] * 9)

    def evict(*sizes, pointers=None, dtype=0):
        return handle.gdn2_evict_tokens(*(pointers or [one] * 8), 2, 2, *sizes, dtype, null)

    good = [1, 4, 16, 1, 64, 2, 2, 16, 0, 0]   # batch, pages, page, heads, dim, columns, new columns, keep, sinks, recent
    assert evict(*good, pointers=[null] + [one] * 7) == -1 and evict(*good, dtype=7) == -3
    for i in range(7):
        assert evict(*[0 if j == i else x for j, x in enumerate(good)]) == -2
    assert evict(*good[:7], 33, 0, 0) == evict(*good[:7], 0, 0, 0) == evict(*good[:7], 16, 9, 8) == evict(*good[:7], 16, -1, 0) == -4
    assert evict(*good, pointers=[ctypes.c_void_p(257)] + [one] * 7) == -5
    assert evict(1, 4, 2 ** 30, 1, 64, 2, 2, 16, 0, 0) == -9
    assert handle.gdn2_evict_workspace_bytes(2, 3, 10) >= 2 * 3 * 11 * 4 and handle.gdn2_evict_workspace_bytes(0, 3, 10) == -2

    def step(batch=1, tokens=1, heads=2, kv_heads=1, dim=64, pages=4, page=16, columns=2, dtype=0, pointers=None):
        return handle.gdn2_weighed_token_attention(*(pointers or [one] * 11), strides, 2, batch, tokens, heads, kv_heads, dim, pages, page,
                                                   columns, 1.0, dtype, 1.0, null)

    assert step(pointers=[one] * 5 + [null] + [one] * 5) == -1
    assert step(batch=0) == step(tokens=0) == step(heads=3, kv_heads=2) == step(dim=60) == step(pages=0) == step(columns=0) == -2
    assert step(dtype=2) == -3 and step(tokens=129) == -9 and step(page=2 ** 30) == -9
    assert step(pointers=[ctypes.c_void_p(264)] + [one] * 10) == -5
    assert handle.gdn2_weighed_token_workspace_bytes(1, 129, 2, 1, 64, 16, 2) == -9
    assert handle.gdn2_attention_weights(*[one] * 2, null, one, null, strides, null, 1, 8, 1, 1, 64, 0, 1.0, null) == -1
    assert handle.gdn2_attention_weights(*[one] * 4, null, strides, null, 1, 8, 1, 1, 60, 0, 1.0, null) == -2
    assert handle.gdn2_attention_weights_bytes(null, 0, 8, 1, 1) == -2
    assert handle.gdn2_window_tree_attention(*[one] * 8, null, *[one] * 2, strides, 2, 0, 0, 1, 1, 2, 1, 64, 4, 16, 2, 8, 0, 0, 1.0, null) == -4   # a mask without depths
