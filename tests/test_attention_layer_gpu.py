"""GPU tests of the attention operators together (examples/attention_layer.py), and of the native host path against the
Python one."""

from __future__ import annotations

import pathlib
import sys

import pytest
import torch

from gdn2_sm120_b200 import _lib
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen
from gdn2_sm120_b200.paged import append_tokens, tree_attention
from gdn2_sm120_b200.rotary import apply_rotary, rotary_tables

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "examples"))

import attention_layer as example

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_drafted_tokens_get_what_one_prompt_gives():
    got, tokens, layer = example.serve(prompt_tokens=150, rounds=8)
    q, k, v = layer.project(tokens, None)
    want = causal_attention(q, k, v).flatten(-2) @ layer.w_out
    assert got.shape == want.shape == (1, 150 + 2 * (3 + 2 + 1 + 1), 256)
    # two roundings of weights and outputs (2^-8 each, independent) through one product, in the norm of all tokens
    assert (got - want).float().norm() <= 2.0 ** -7 * want.float().norm()


def test_a_training_step_of_both_kinds_of_layers():
    loss, grads = example.training_step()
    again, same = example.training_step()
    assert torch.isfinite(loss) and loss == again
    assert all(torch.isfinite(g).all() and g.any() for g in grads) and all(torch.equal(a, b) for a, b in zip(grads, same))


def _everything():
    gen = torch.Generator(device=DEV).manual_seed(0)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV).bfloat16()

    q, k, v, do = normal(1, 200, 4, 64), normal(1, 200, 2, 64), normal(1, 200, 2, 64), normal(1, 200, 4, 64)
    cos, sin = rotary_tables(200, 32)
    positions = torch.arange(200, device=DEV)[None]
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    turned = apply_rotary(*leaves[:2], cos, sin, positions, layout="interleaved")
    out = causal_attention_varlen(*turned, leaves[2], (0, 3, 130, 200), scale=0.2)
    results = [out.detach(), *torch.autograd.grad(out, leaves, do)]
    results += [causal_attention(q, k, v), *apply_rotary(q, k, cos, sin)]
    pages = [normal(9, 16, 2, 64) for _ in range(2)]
    slots = torch.randperm(144, generator=gen, device=DEV)[:100]
    append_tokens(k[0, :100], v[0, :100], *pages, slots)
    table = torch.randperm(9, generator=gen, device=DEV).int()[None]
    mask = torch.rand(7, 7, generator=gen, device=DEV) < 0.5
    results += [*pages, tree_attention(q[:, :7], k[:, :7], v[:, :7], *pages, table, torch.tensor([133], device=DEV, dtype=torch.int32), mask)]
    return results


def test_native_and_python_host_paths_give_the_same():
    _lib.LAUNCHES[0] = 0
    native = _everything()
    launches = _lib.LAUNCHES[0]
    _lib.LAUNCHES[0] = 0
    _lib.KERNEL_EVENTS = {}      # calls that are timed one by one go through Python
    try:
        python = _everything()
        names = set(_lib.KERNEL_EVENTS)
    finally:
        _lib.KERNEL_EVENTS = None
    assert {"gdn2_rotary", "gdn2_attention_forward", "gdn2_attention_backward", "gdn2_append_tokens", "gdn2_tree_attention"} <= names
    assert launches == _lib.LAUNCHES[0] > 0
    assert all(torch.equal(a, b) for a, b in zip(native, python))
