"""GPU tests of attention over a paged cache where values are not finite: they cost little, and reach the rows that see them in every
unit of a CTA."""

from __future__ import annotations

import math

import pytest
import torch

from gdn2_sm120_b200.eviction import weighed_token_attention
from gdn2_sm120_b200.paged import tree_attention
from gdn2_sm120_b200.window import window_tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _setting(batch, cached, drafted, heads, kv_heads, dim, page, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    columns = -(-(cached + drafted) // page)
    q, k, v = (torch.randn(batch, drafted, h, dim, generator=gen, device=DEV).to(BF16) for h in (heads, kv_heads, kv_heads))
    pages = [torch.randn(batch * columns, page, kv_heads, dim, generator=gen, device=DEV).to(BF16) for _ in range(2)]
    table = torch.randperm(batch * columns, generator=gen, device=DEV).int().view(batch, columns)
    lengths = torch.full((batch,), cached, device=DEV, dtype=torch.int32) - torch.arange(batch, device=DEV, dtype=torch.int32) % 3
    return q, k, v, pages, table, lengths


def _place(table, lengths, b, t, page):
    return table[b, t // page].long(), t % page


def _microseconds(call):
    best = math.inf
    for _ in range(12):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        call()
        end.record()
        torch.cuda.synchronize()
        best = min(best, 1000.0 * start.elapsed_time(end))
    return best


@pytest.mark.parametrize("drafted,heads,kv_heads,window,sinks", [(1, 8, 2, 7000, 4), (1, 32, 8, 4096, 0), (2, 8, 2, 5000, 300), (40, 8, 2, 7000, 4)])
def test_a_value_that_is_not_finite_costs_little(drafted, heads, kv_heads, window, sinks):
    """The whole window is not gone through for it, in the kernel for few rows and in that for many."""

    page = 64
    q, k, v, pages, table, lengths = _setting(16, 9000, drafted, heads, kv_heads, 128, page)
    clean = _microseconds(lambda: window_tree_attention(q, k, v, *pages, table, lengths, window, sinks=sinks))
    strange = v.clone()
    strange[0, 0, 0, 3] = math.nan
    drafts = _microseconds(lambda: window_tree_attention(q, k, strange, *pages, table, lengths, window, sinks=sinks))
    where = _place(table, lengths, 1, int(lengths[1]) - window + 1, page)
    pages[1][where[0], where[1], 0, 3] = math.nan
    edge = _microseconds(lambda: window_tree_attention(q, k, v, *pages, table, lengths, window, sinks=sinks))
    # a look at few tokens for every unit; the window's tokens one after the other are milliseconds
    assert max(drafts, edge) < 2.0 * clean + 100.0, f"{clean:.0f} us, with NaN {drafts:.0f} and {edge:.0f}"


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cached,drafted,heads,kv_heads,window,sinks", [
    (5000, 1, 8, 4, 4500, 0), (5000, 3, 4, 4, 4500, 70), (3000, 4, 8, 2, 2900, 4), (2500, 5, 24, 8, 400, 4), (5000, 20, 8, 4, 4500, 70), (3000, 70, 4, 2, 2100, 4),
    (700, 30, 16, 2, 3, 0),
])
def test_values_at_the_edge_and_drafted_in_many_units(what, cached, drafted, heads, kv_heads, window, sinks):
    """Several units a CTA, tokens that are a multiple of 2048 apart, a deep tree whose tokens lose sight of many cached ones."""

    batch, page, dim = 20, 16, 64
    q, k, v, pages, table, lengths = _setting(batch, cached, drafted, heads, kv_heads, dim, page, seed=drafted)
    mask = torch.ones(drafted, drafted, device=DEV, dtype=torch.bool).tril()
    for depths in (torch.arange(drafted, device=DEV, dtype=torch.int32), torch.arange(drafted, device=DEV, dtype=torch.int32) * 97):
        clean = window_tree_attention(q, k, v, *pages, table, lengths, window, mask, depths, sinks=sinks)
        values, drafts = pages[1].clone(), v.clone()
        reached = torch.zeros_like(clean, dtype=torch.bool)
        group = heads // kv_heads
        for b in range(0, batch, 2):
            n = int(lengths[b])
            place = n + depths.long()
            cached_ones = {n - window + 1, n - window + 2, n - window + 40, n - 1, n - 2049, sinks - 1, sinks, n - window + 1 + int(depths[-1])}
            for t in {t for t in cached_ones if 0 <= t < n}:
                head, channel = (b + t) % kv_heads, (5 * t + b) % dim
                where = _place(table, lengths, b, t, page)
                values[where[0], where[1], head, channel] = what
                sees = (place - t < window) | (t < sinks)
                reached[b, :, head * group:(head + 1) * group, channel] |= sees[:, None]
            for d in {0, drafted // 2, drafted - 1}:
                head, channel = (b + d) % kv_heads, (3 * d + b) % dim
                drafts[b, d, head, channel] = what
                sees = mask[:, d] & ((place - place[d] < window) | (place[d] < sinks))
                reached[b, :, head * group:(head + 1) * group, channel] |= sees[:, None]
        out = window_tree_attention(q, k, drafts, pages[0], values, table, lengths, window, mask, depths, sinks=sinks)
        assert torch.equal(out[~reached], clean[~reached])
        assert not torch.isfinite(out[reached]).any()


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_new_values_of_many_rows_with_weights(what):
    """Blocks of 16 rows: a new token's value reaches the tokens behind it, in every block, and no weight."""

    batch, drafted, heads, kv_heads, page = 6, 40, 8, 2, 16
    q, k, v, pages, table, lengths = _setting(batch, 300, drafted, heads, kv_heads, 64, page, seed=3)
    weights = torch.rand(pages[0].shape[0], kv_heads, page, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    places = lengths.long()[:, None] + torch.arange(drafted, device=DEV)
    slots = table.long().gather(1, places // page) * page + places % page
    kept = weights.clone()
    clean = weighed_token_attention(q, k, v, *pages, kept, table, lengths, slots)
    strange = v.clone()
    reached = torch.zeros_like(clean, dtype=torch.bool)
    for b in range(0, batch, 2):
        for d in (0, 5, 17, 39):
            head, channel = (b + d) % 2, (11 * d + b) % 64
            strange[b, d, head, channel] = what
            reached[b, d:, head * 4:(head + 1) * 4, channel] = True
    out = weighed_token_attention(q, k, strange, *pages, weights, table, lengths, slots)
    assert torch.equal(out[~reached], clean[~reached]) and not torch.isfinite(out[reached]).any()
    assert torch.equal(weights, kept)
    # (a step without weights meets the same values)
    without = tree_attention(q, k, strange, *pages, table, lengths)
    assert torch.equal(torch.isfinite(without), torch.isfinite(out))
