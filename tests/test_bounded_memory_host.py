"""Host-side checks of the operators of bounded memory that need no GPU: what refusals say."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from gdn2_sm120_b200.attention import causal_attention
from gdn2_sm120_b200.eviction import weighed_attention
from gdn2_sm120_b200.window import window_attention, window_attention_varlen

Q, K = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)


def test_forward_mode_tangents_are_refused_by_name():
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(K.clone(), torch.ones_like(K))
        for call, name in ((lambda: causal_attention(Q, dual, K), "causal attention"), (lambda: window_attention(Q, dual, K, 2), "attention with a window"),
                           (lambda: window_attention_varlen(Q, K, dual, (0, 4), 2), "attention with a window"),
                           (lambda: weighed_attention(Q, dual, K), "weighed_attention")):
            with pytest.raises(RuntimeError, match=f"^{name} has no forward-mode"):
                call()
