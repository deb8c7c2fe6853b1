"""Host-side checks of attention with a window that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gdn2_sm120_b200 import _lib
from gdn2_sm120_b200.window import window_attention, window_attention_varlen

Q, K = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)


def test_tensors_on_the_cpu_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        window_attention(Q, K, K, 2)
    with pytest.raises(ValueError, match="CUDA"):
        window_attention_varlen(Q, K, K, (0, 4), 2, sinks=1)


@pytest.mark.parametrize("window,sinks,error", [
    (0, 0, ValueError), (-3, 0, ValueError), (2, -1, ValueError), (2.0, 0, TypeError), (None, 0, TypeError), (True, 0, TypeError),
    (torch.tensor(2), 0, TypeError), (2, 1.0, TypeError), (2, None, TypeError), ("2", 0, TypeError),
])
def test_windows_that_are_none(window, sinks, error):
    with pytest.raises(error):
        window_attention(Q, K, K, window, sinks=sinks)
    with pytest.raises(error):
        window_attention_varlen(Q, K, K, (0, 4), window, sinks=sinks)


def test_entry_points_reject_bad_windows_without_a_gpu():
    handle, one = _lib.lib(), ctypes.c_void_p(256)
    strides = _lib.int64s(*[64] * 12)
    for window, sinks in ((0, 0), (-1, 0), (1, -1)):
        assert handle.gdn2_window_attention_forward(*[one] * 4, None, None, strides, None, 1, 8, 1, 1, 64, window, sinks, 0, 1.0, None) == -4
        assert handle.gdn2_window_attention_backward(*[one] * 11, strides, None, 1, 8, 1, 1, 64, window, sinks, 0, 1.0, None) == -4
        assert handle.gdn2_window_attention_backward_bytes(None, 1, 8, 1, 1, 64, window, sinks) == -4
    assert handle.gdn2_window_attention_forward(*[None] * 6, strides, None, 1, 8, 1, 1, 64, 4, 0, 0, 1.0, None) == -1
    assert handle.gdn2_window_attention_forward(*[one] * 4, None, None, strides, None, 1, 8, 1, 1, 60, 4, 0, 0, 1.0, None) == -2
    assert handle.gdn2_window_attention_forward(*[one] * 4, None, None, strides, None, 1, 8, 1, 1, 64, 4, 0, 2, 1.0, None) == -3
