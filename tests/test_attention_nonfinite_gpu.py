"""GPU tests of causal attention with values that are not finite in long prompts and many work items: they change the
channels and rows that see them, and not one bit of anything else."""

from __future__ import annotations

import math

import pytest
import torch

import attention_bounds as exact
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(batch, time, heads, kv_heads, dim, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(batch, time, h, dim, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads, kv_heads)]


def _check(q, k, v, bounds, places):
    """places: (batch entry, row, key head, channel, value); compared with the call in which all values are finite."""

    batch, total, heads, dim = q.shape
    group = heads // k.shape[2]

    def run(v):
        return causal_attention(q, k, v) if bounds is None else causal_attention_varlen(q, k, v, bounds)

    clean = run(v)
    v = v.clone()
    reached = torch.zeros(batch, total, heads, dim, device=DEV, dtype=torch.bool)
    nan = torch.zeros_like(reached)
    for b, row, head, channel, value in places:
        v[b, row, head, channel] = value
        end = total if bounds is None else next(x for x in bounds if x > row)
        at = (b, slice(row, end), slice(head * group, (head + 1) * group), channel)
        reached[at] = True
        nan[at] |= math.isnan(value)
    out = run(v)
    assert torch.equal(out[~reached], clean[~reached])
    assert not torch.isfinite(out[reached]).any() and torch.isnan(out[nan]).all()


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("time,row", [(16300, 16290), (16384, 16383), (16300, 16127)])
def test_one_value_late_in_a_long_prompt(value, time, row):
    """Up to 127 rows before it meet it in their tile."""

    _check(*_inputs(1, time, 4, 2, 128, BF16), None, [(0, row, 1, 77, value)])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_one_value_late_in_a_long_packed_prompt(dtype):
    q, k, v = _inputs(1, 16700, 4, 1, 64, dtype)
    _check(q, k, v, (0, 130, 16130, 16700), [(0, 16129, 0, 5, math.nan), (0, 129, 0, 63, math.inf)])


@pytest.mark.parametrize("dim", [40, 64, 96, 128])
def test_values_in_many_items_of_a_cta(dim):
    """8 x 3 x 32 items: several a CTA are done once more, in tiles of either query tile, at their ends and beginnings."""

    places = [(b, row, (b + row) % 8, (7 * row) % dim, (math.nan, math.inf, -math.inf)[row % 3])
              for b in range(0, 8, 2) for row in (0, 1, 127, 128, 200, 255, 256, 511, 512, 640, 699)]
    _check(*_inputs(8, 700, 32, 8, dim, FP16), None, places)


def test_values_in_short_packed_prompts():
    lengths = [1, 5, 64, 127, 128, 129, 200, 255, 256, 257, 300, 2, 90, 31] * 4
    bounds = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    places = [(0, lo + (n - 1) * (i % 3) // 2, i % 2, i % 128, math.inf if i % 2 else math.nan)
              for i, (lo, n) in enumerate(zip(bounds, lengths)) if i % 5]
    _check(*_inputs(1, bounds[-1], 8, 2, 128, BF16), bounds, places)


def test_whole_rows_of_padding():
    """The end of every sequence of a batch is padding that holds anything."""

    q, k, v = _inputs(4, 900, 8, 2, 128, BF16)
    clean = causal_attention(q, k, v)
    used = (900, 773, 130, 1)
    for b, n in enumerate(used):
        for x, value in ((q, math.nan), (k, math.inf), (v, math.nan)):
            x[b, n:] = value
    out = causal_attention(q, k, v)
    for b, n in enumerate(used):
        assert torch.equal(out[b, :n], clean[b, :n])
        assert torch.isnan(out[b, n:]).all()


def test_inf_and_minus_inf_that_a_row_sees_both():
    q, k, v = _inputs(1, 300, 2, 1, 64, BF16)
    v[0, 10, 0, 3], v[0, 200, 0, 3], v[0, 290, 0, 3] = math.inf, math.inf, -math.inf
    out = causal_attention(q, k, v)[0, :, :, 3]
    assert torch.isfinite(out[:10]).all() and torch.isposinf(out[10:290]).all() and torch.isnan(out[290:]).all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("time,at", [(700, 300), (700, 0), (700, 383), (130, 129)])
def test_gradients_of_rows_that_do_not_see_it(which, value, time, at):
    """A value that is not finite makes the gradients of what it is part of not finite: its own row, the rows that see it and
    the keys that those see.  Beyond that, a key reaches dq, in its channel, of the rows before it in its tile of 128 tokens; a
    query reaches dk, and a cotangent dv, of the keys behind it in its tile.  Everything else is as it was: to the bit where
    no score is infinite (one that is lets the rows of its tile look for their maxima more often, which rounds differently)."""

    channel, head, kv_head = 5, 1, 0
    q, k, v = _inputs(1, time, 4, 2, 64, BF16, seed=3)
    do = _inputs(1, time, 4, 2, 64, BF16, seed=4)[0]
    tensors = dict(q=q, k=k, v=v, do=do)

    def run():
        leaves = [tensors[x].detach().requires_grad_(True) for x in "qkv"]
        out = causal_attention(*leaves)
        return dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, tensors["do"])))

    clean = run()
    tensors[which] = tensors[which].clone()
    tensors[which][0, at, head if which in ("q", "do") else kv_head, channel] = value
    got = run()
    tile = slice(at // 128 * 128, at // 128 * 128 + 128)
    may = {x: torch.zeros_like(y, dtype=torch.bool) for x, y in clean.items()}
    if which in ("q", "do"):       # row `at` of head 1, and what it sees
        may["dq"][0, at, head] = True
        may["dk"][0, :at + 1, kv_head] = may["dv"][0, :at + 1, kv_head] = True
        may["dk" if which == "q" else "dv"][0, tile, kv_head, channel] = True
    else:                           # every row from `at` on of the heads 0 and 1, and what those see
        may["dq"][0, at:, :2] = True
        may["dk"][0, :, kv_head] = may["dv"][0, :, kv_head] = True
        if which == "k":
            may["dq"][0, tile, :2, channel] = True
    want = exact.attention(*(x[0].transpose(0, 1) for x in (q, k, v)), exact.causal(time, DEV), 64 ** -0.5, do[0].transpose(0, 1))
    for x in clean:
        untouched = ~may[x]
        if math.isnan(value) or which in ("v", "do"):
            assert torch.equal(got[x][untouched], clean[x][untouched]), x
        off, bound = (got[x][0].double() - want[x][0].transpose(0, 1)).abs(), want[x][1].transpose(0, 1)
        assert (off <= bound)[untouched[0]].all(), x
    if math.isnan(value):           # (a score of -inf, or values alone, leave the weights that dv is made of finite)
        assert torch.isnan(got["dk" if which == "v" else "dv"][0, at, kv_head, channel])
