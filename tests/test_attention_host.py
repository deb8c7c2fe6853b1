"""Host-side checks of the attention layer's operators that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gdn2_sm120_b200 import _lib, _validate
from gdn2_sm120_b200.attention import _launches, causal_attention, causal_attention_varlen
from gdn2_sm120_b200.paged import append_tokens, tree_attention
from gdn2_sm120_b200.rotary import apply_rotary, rotary_tables


def test_tensors_on_the_cpu_are_refused():
    q, k = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    cos, sin = rotary_tables(4, 64, device="cpu")
    pages = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        causal_attention(q, k, k)
    with pytest.raises(ValueError, match="CUDA"):
        causal_attention_varlen(q, k, k, (0, 4))
    with pytest.raises(ValueError, match="CUDA"):
        apply_rotary(q, k, cos, sin)
    with pytest.raises(ValueError, match="CUDA"):
        append_tokens(k, k, pages, pages.clone(), torch.zeros(1, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        tree_attention(q, k, k, pages, pages.clone(), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("args,kwargs", [
    ((0, 64), {}), ((4, 63), {}), ((4, 0), {}), ((4, 64), dict(scaling="other")), ((4, 64), dict(factor=0.5)), ((4, 64), dict(base=0.0)),
    ((4, 64), dict(scaling="yarn", factor=2.0)), ((4, 64), dict(scaling="yarn", factor=2.0, trained=0)),
    ((4, 64), dict(scaling="yarn", factor=2.0, trained=9, fast=1.0, slow=1.0)), ((4, 2), dict(scaling="ntk", factor=2.0)), ((True, 64), {}),
    ((4, 64), dict(factor=float("nan"))),
])
def test_tables_refuse(args, kwargs):
    with pytest.raises(ValueError):
        rotary_tables(*args, **kwargs, device="cpu")


def test_statistics_are_padded_to_tiles_per_sequence():
    rows = _lib.lib().gdn2_attention_stat_rows
    assert rows(None, 3, 257) == 3 * 512
    assert rows(_lib.int64s(0, 0, 1, 257, 600), 4, 600) == 256 + 256 + 512
    assert rows(_lib.int64s(0, 5, 4), 2, 5) < 0 and rows(_lib.int64s(0, 9), 1, 5) < 0 and rows(None, 0, 5) < 0


def test_launch_counts_of_packed_calls():
    assert _launches(None) == 1
    assert _launches((0, 5)) == 1 and _launches((0, 0, 0)) == 0
    assert _launches(tuple(range(257))) == 1 and _launches(tuple(range(258))) == 2
    assert _launches((0,) * 257 + (4,)) == 1


def test_extent_and_strides_of_views():
    x = torch.zeros(2, 6, 4, 8, dtype=torch.bfloat16)
    lo = x.data_ptr()
    assert _validate.extent(x) == (lo, lo + x.numel() * 2)
    assert _validate.extent(x[:, 1:3, :2]) == (lo + 64, lo + 64 + (192 + 32 + 8 + 7 + 1) * 2)
    begin, end = _validate.extent(x[:0])
    assert begin == end
    assert _validate.head_strides(x) == (192, 32, 8)
    assert _validate.head_strides(x[:1, :, :1].as_strided((1, 6, 1, 8), (7, 32, 3, 1))) == (48, 32, 8)


def test_entry_points_check_their_arguments():
    handle, buffer = _lib.lib(), (ctypes.c_char * 4096)()
    at = (ctypes.addressof(buffer) + 63) // 64 * 64
    strides = _lib.int64s(*([64, 64, 64] * 4))

    def forward(q=at, heads=2, kv_heads=1, dim=64, dtype=0, time=4, strides=strides):
        return handle.gdn2_attention_forward(q, at, at, at, None, strides, None, 1, time, heads, kv_heads, dim, dtype, 1.0, None)

    assert forward(q=None) == -1 and forward(q=at + 2) == -5 and forward(strides=_lib.int64s(*([64, 64, 4] * 3))) == -5
    assert forward(heads=3, kv_heads=2) == -2 and forward(dim=60) == -2 and forward(dim=136) == -2 and forward(time=0) == -2
    assert forward(dtype=2) == -3 and forward(time=2 ** 40) < 0

    def rotary(dim=64, pairs=32, dtype=0, cos=at, time=1):
        return handle.gdn2_rotary(at, at, at, at, cos, at, None, strides, 0, 1, time, 1, 1, dim, pairs, 4, 0, 0, dtype, None)

    assert rotary(cos=None) == -1 and rotary(pairs=33) == -2 and rotary(dim=514) == -2 and rotary(dtype=3) == -3 and rotary(time=0) == -2
    assert rotary(cos=at + 2) == -5

    def append(tokens=1, slots=at, dtype=0, pages=1):
        return handle.gdn2_append_tokens(at, at, at, at, slots, strides, tokens, pages, 16, 1, 8, dtype, None)

    assert append(slots=None) == -1 and append(tokens=0) == -2 and append(dtype=7) == -3 and append(slots=at + 4) == -5 and append(pages=2 ** 40) == -9

    def tree(drafted=1, table=at, dim=64, page=16, columns=1, workspace=at):
        return handle.gdn2_tree_attention(at, at, at, at, at, table, at, None, at, workspace, strides, 1, 0, 1, drafted, 2, 1, dim, 1, page,
                                          columns, 0, 1.0, None)

    assert tree(table=None) == -1 and tree(drafted=0) == -2 and tree(dim=12) == -2 and tree(workspace=at + 4) == -5
    assert tree(page=2 ** 20, columns=2 ** 12) == -9
    assert handle.gdn2_tree_workspace_bytes(1, 3, 2, 64) == -2


def test_tree_attention_refuses_more_tokens_than_31_bits_number():
    handle, buffer = _lib.lib(), (ctypes.c_char * 4096)()
    at = (ctypes.addressof(buffer) + 63) // 64 * 64
    strides = _lib.int64s(*([64] * 9))

    def tree(drafted, columns):
        return handle.gdn2_tree_attention(at, at, at, at, at, at, at, None, at, at, strides, 1, 0, 1, drafted, 2, 1, 64, 1, 16, columns, 0,
                                          1.0, None)

    # each side alone would fit an int, both together would not
    assert tree(drafted=2 ** 29, columns=2 ** 26) == -9
    assert tree(drafted=1, columns=2 ** 26) == -9 and tree(drafted=2 ** 30, columns=1) == -9


def test_forward_mode_tangents_are_refused():
    """They would be dropped in silence: no kernel has a forward-mode derivative."""

    from torch.autograd import forward_ad

    q, k = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    cos, sin = rotary_tables(4, 64, device="cpu")
    pages = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    calls = (lambda x: causal_attention(q, x, k), lambda x: causal_attention_varlen(q, k, x, (0, 4)), lambda x: apply_rotary(q, x, cos, sin),
             lambda x: apply_rotary(q, x, cos, sin, inplace=True), lambda x: append_tokens(x, k, pages, pages.clone(), torch.zeros(1, 4).long()),
             lambda x: tree_attention(q, x, k, pages, pages.clone(), table, lengths))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(k.clone(), torch.ones_like(k))
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
            with pytest.raises(ValueError, match="CUDA"):      # no tangent: the usual refusal of this test's tensors
                call(k)
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call(k)
