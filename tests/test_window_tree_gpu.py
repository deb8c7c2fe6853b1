"""GPU tests of attention with a window and sinks over a paged cache, against plain attention in 64 bits within bounds that
follow from what the kernels round (tests/attention_bounds.py)."""

from __future__ import annotations

import math

import pytest
import torch

import attention_bounds as exact
from gdn2_sm120_b200.paged import append_tokens, tree_attention
from gdn2_sm120_b200.window import window_attention, window_tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _cache(lengths, page, kv_heads, dim, dtype, seen=None, seed=0):
    """Pages in no order.  `seen(b, n)`: which of a sequence's tokens some row sees; all other places hold NaN, and pages
    without such a token have entries that name no page."""

    gen = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages, columns = sum(need) + 3, max(1, *need)
    k, v = (torch.randn(pages, page, kv_heads, dim, generator=gen, device=DEV).to(dtype) for _ in range(2))
    order = torch.randperm(pages, generator=gen, device=DEV).int()
    table = torch.full((len(lengths), columns), -5, device=DEV, dtype=torch.int32)
    used = torch.zeros(pages, page, device=DEV, dtype=torch.bool)
    at = 0
    for b, (n, count) in enumerate(zip(lengths, need)):
        table[b, :count] = order[at:at + count]
        at += count
        t = torch.arange(n, device=DEV)
        there = t >= 0 if seen is None else seen(b, n)
        used[table[b, t // page].long()[there], (t % page)[there]] = True
        columns_used = torch.zeros(count, device=DEV, dtype=torch.bool)
        columns_used[(t // page)[there]] = True
        table[b, :count][~columns_used] = -7 if b % 2 else 10 ** 9
    k[~used], v[~used] = math.nan, math.nan
    return k, v, table, torch.tensor(lengths, device=DEV, dtype=torch.int32)


def _fresh(batch, drafted, heads, kv_heads, dim, dtype, seed=1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(batch, drafted, h, dim, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads, kv_heads)]


def _tree(batch, drafted, seed=2):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    mask = torch.eye(drafted, device=DEV, dtype=torch.bool).repeat(batch, 1, 1)
    for b in range(batch):
        for i in range(1, drafted):
            mask[b, i] |= mask[b, int(torch.randint(0, i, (), generator=gen, device=DEV))]
    return mask, mask.sum(-1, dtype=torch.int32) - 1


def _seen(n, drafted, window, sinks, mask, depths):
    """[drafted, n + drafted]"""

    depths = depths.long().clamp_min(0)
    place = torch.cat([torch.arange(n, device=DEV), n + depths])
    seen = torch.cat([torch.ones(drafted, n, device=DEV, dtype=torch.bool), mask], 1)
    return seen & (((n + depths)[:, None] - place < window) | (place < sinks))


def _check(out, q, k, v, cache, window, sinks, mask, depths, scale=None):
    k_pages, v_pages, table, lengths = cache
    page, drafted, dim = k_pages.shape[1], q.shape[1], q.shape[3]
    for b in range(q.shape[0]):
        n = int(lengths[b])
        t = torch.arange(n, device=DEV)
        seen = _seen(n, drafted, window, sinks, mask if mask.ndim == 2 else mask[b], depths if depths.ndim == 1 else depths[b])
        pages = table[b, t // page].long()
        pages[~seen[:, :n].any(0)] = 0
        keys, values = (torch.cat([torch.where(seen[:, :n].any(0)[:, None, None], x[pages, t % page], 0), y[b]])
                        for x, y in ((k_pages, k), (v_pages, v)))
        want = exact.attention(*(x.transpose(0, 1) for x in (q[b], keys, values)), seen, dim ** -0.5 if scale is None else scale)
        exact.check(f"sequence {b}", out[b], *want["o"])


def _chain(drafted):
    return torch.ones(drafted, drafted, device=DEV, dtype=torch.bool).tril(), torch.arange(drafted, device=DEV, dtype=torch.int32)


CASES = [
    ((0,), 16, 1, 1, 1, 128, 1, 0), ((1, 0, 15, 16, 17), 16, 1, 4, 1, 64, 1, 0), ((1, 0, 15, 16, 17), 16, 1, 4, 1, 64, 2, 1),
    ((63, 640, 65), 64, 1, 8, 8, 128, 64, 2), ((500, 3), 24, 2, 6, 2, 96, 100, 4), ((129, 1000), 7, 5, 8, 2, 128, 130, 0),
    ((300, 1300), 128, 7, 16, 2, 128, 128, 128), ((1040, 260, 0), 16, 16, 2, 1, 8, 257, 300), ((64, 128, 777), 32, 33, 4, 2, 72, 20, 1),
    ((200, 900), 1, 48, 8, 1, 64, 3, 130), ((470,), 16, 64, 2, 2, 128, 129, 4), ((5, 400), 16, 65, 3, 1, 128, 7, 0),
    ((700,), 48, 130, 2, 1, 40, 256, 64), ((2000, 130), 64, 20, 16, 1, 128, 385, 2000), ((2500,) * 9, 32, 4, 4, 2, 64, 1111, 5),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,page,drafted,heads,kv_heads,dim,window,sinks", CASES)
def test_trees_over_a_cache(dtype, lengths, page, drafted, heads, kv_heads, dim, window, sinks):
    q, k, v = _fresh(len(lengths), drafted, heads, kv_heads, dim, dtype)
    for mask, depths in (_tree(len(lengths), drafted), _chain(drafted)):
        def seen(b, n):
            return _seen(n, drafted, window, sinks, *(x if x.ndim == d else x[b] for x, d in ((mask, 2), (depths, 1))))[:, :n].any(0)

        cache = _cache(lengths, page, kv_heads, dim, dtype, seen)
        out = window_tree_attention(q, k, v, *cache, window, mask, depths, sinks=sinks)
        assert out.shape == q.shape and out.is_contiguous()
        _check(out, q, k, v, cache, window, sinks, mask, depths)
    plain = window_tree_attention(q, k, v, *cache, window, sinks=sinks)
    assert torch.equal(plain, out) and torch.equal(plain, window_tree_attention(q, k, v, *cache, window, None, depths, sinks=sinks))


@pytest.mark.parametrize("drafted,heads", [(1, 4), (3, 8), (20, 4), (40, 16)])
def test_a_window_over_everything_is_tree_attention(drafted, heads):
    lengths = (700, 0, 90)
    cache = _cache(lengths, 16, 2, 64, BF16)
    q, k, v = _fresh(3, drafted, heads, 2, 64, BF16)
    mask, depths = _tree(3, drafted)
    want = tree_attention(q, k, v, *cache, mask)
    for window, sinks in ((741, 0), (2 ** 50, 9), (1, 800), (1, 2 ** 40)):
        assert torch.equal(window_tree_attention(q, k, v, *cache, window, mask, depths, sinks=sinks), want)


def test_decoding_gives_what_one_prompt_gives():
    """Tokens one by one, and three at a time, over a cache that they are appended to."""

    time, window, sinks, page = 333, 70, 3, 16
    q, k, v = _fresh(1, time, 4, 2, 64, BF16)
    want = window_attention(q, k, v, window, sinks=sinks)
    table = torch.randperm(21, device=DEV).int()[None]
    for step in (1, 3):
        pages = [torch.full((21, page, 2, 64), math.nan, device=DEV, dtype=BF16) for _ in range(2)]
        length = torch.zeros(1, device=DEV, dtype=torch.int32)
        for at in range(0, time, step):
            now = slice(at, at + step)
            out = window_tree_attention(q[:, now], k[:, now], v[:, now], *pages, table, length, window, sinks=sinks)
            place = torch.arange(at, at + step, device=DEV)
            append_tokens(k[0, now], v[0, now], *pages, table[0, place // page].long() * page + place % page)
            length += step
            # two roundings of weights and outputs each
            assert (out - want[:, now]).float().norm() <= 2.0 ** -6 * want[:, now].float().norm()


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("drafted,heads", [(3, 2), (3, 8), (20, 4), (40, 16)])
def test_cached_values_that_some_rows_do_not_see(what, drafted, heads):
    """reach those that see them, and not one bit of the others."""

    lengths, window, sinks, page = (600, 300, 5), 100, 4, 16
    cache = _cache(lengths, page, 2, 64, FP16)
    q, k, v = _fresh(3, drafted, heads, 2, 64, FP16)
    mask, depths = _tree(3, drafted)
    clean = window_tree_attention(q, k, v, *cache, window, mask, depths, sinks=sinks)
    for b, t in ((0, 501), (0, 502), (0, 500), (0, 2), (1, 202), (1, 299), (2, 4)):
        values = cache[1].clone()
        values[cache[2][b, t // page].long(), t % page, 1, 9] = what
        out = window_tree_attention(q, k, v, cache[0], values, *cache[2:], window, mask, depths, sinks=sinks)
        reached = torch.zeros_like(out, dtype=torch.bool)
        reached[b, :, heads // 2:, 9] = _seen(lengths[b], drafted, window, sinks, mask[b], depths[b])[:, t, None]
        assert torch.equal(out[~reached], clean[~reached])
        assert not torch.isfinite(out[reached]).any()


@pytest.mark.parametrize("drafted", [4, 30])
def test_drafted_values_that_some_rows_do_not_see(drafted):
    cache = _cache((200,), 16, 1, 64, BF16)
    q, k, v = _fresh(1, drafted, 4, 1, 64, BF16)
    window, (mask, depths) = 2, _chain(drafted)
    clean = window_tree_attention(q, k, v, *cache, window)
    v[0, 1, 0, 3] = math.inf
    out = window_tree_attention(q, k, v, *cache, window)
    rows = [i for i in range(drafted) if i not in (1, 2)]
    assert torch.equal(out[:, rows], clean[:, rows])
    assert torch.isposinf(out[:, 1:3, :, 3]).all()


def test_depths_of_any_size():
    """Negative ones count as 0; a deep token sees no cached ones but the sinks."""

    cache = _cache((500,), 16, 2, 64, BF16)
    q, k, v = _fresh(1, 6, 4, 2, 64, BF16)
    mask = torch.eye(6, device=DEV, dtype=torch.bool)
    depths = torch.tensor([-5, 0, 90, 100, 2 ** 30 - 1, 2 ** 31 - 1], device=DEV, dtype=torch.int32)
    for sinks in (0, 3):
        out = window_tree_attention(q, k, v, *cache, 100, mask, depths, sinks=sinks)
        _check(out, q, k, v, cache, 100, sinks, mask, depths.clamp(max=2 ** 30 - 1))
    assert torch.equal(window_tree_attention(q, k, v, *cache, 100, mask, depths)[0, 4:], v[0, 4:].repeat_interleave(2, 1))


def test_many_sequences_and_a_long_one():
    lengths = [(37 * i) % 900 for i in range(300)] + [30011]
    cache = _cache(lengths, 16, 1, 64, BF16)
    q, k, v = _fresh(301, 1, 2, 1, 64, BF16)
    mask, depths = _chain(1)
    for window, sinks in ((200, 2), (20000, 500)):
        _check(window_tree_attention(q, k, v, *cache, window, sinks=sinks), q, k, v, cache, window, sinks, mask, depths)


def test_rows_that_see_nothing_give_zero():
    cache = _cache((0, 0, 300), 16, 2, 64, BF16)
    q, k, v = _fresh(3, 6, 4, 2, 64, BF16)
    mask = torch.zeros(3, 6, 6, device=DEV, dtype=torch.bool)
    mask[0, 1, 4] = mask[2, 5, 0] = True
    depths = torch.tensor([0, 1, 2, 3, 4, 60], device=DEV, dtype=torch.int32)
    out = window_tree_attention(q, k, v, *cache, 50, mask, depths)
    _check(out, q, k, v, cache, 50, 0, mask, depths)
    assert not out[0, 0].any() and not out[1].any() and not out[2, 5].any() and out[0, 1].any() and out[2, 0].any()


def test_bad_pages_and_lengths_make_their_sequence_nan():
    lengths = (300, 300, 300, 300)
    for drafted in (1, 20):
        k_pages, v_pages, table, length = _cache(lengths, 16, 2, 64, BF16)
        q, k, v = _fresh(4, drafted, 4, 2, 64, BF16)
        clean = window_tree_attention(q, k, v, k_pages, v_pages, table, length, 100, sinks=4)
        table[1, 15] = k_pages.shape[0]
        length[2], length[3] = -1, table.shape[1] * 16 + 1
        out = window_tree_attention(q, k, v, k_pages, v_pages, table, length, 100, sinks=4)
        assert torch.equal(out[0], clean[0]) and torch.isnan(out[1:]).all()


def test_a_captured_step_with_other_lengths_pages_and_depths():
    cache = _cache((900, 500), 16, 2, 64, BF16)
    q, k, v = _fresh(2, 5, 4, 2, 64, BF16)
    mask, depths = _tree(2, 5)
    window_tree_attention(q, k, v, *cache, 100, mask, depths, sinks=3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_tree_attention(q, k, v, *cache, 100, mask, depths, sinks=3)
    for seed in (5, 6):
        new, depth = _tree(2, 5, seed)
        mask.copy_(new)
        depths.copy_(depth)
        cache[3].sub_(77 * seed)
        cache[2][1] = cache[2][1].roll(1)
        cache[2][1, :10].clamp_(min=0)
        graph.replay()      # (at last the second length is below 0: NaN, in a replayed graph too)
        want = window_tree_attention(q, k, v, *cache, 100, mask, depths, sinks=3)
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(0.0), want.nan_to_num(0.0))


def test_refusals():
    cache = _cache((40,), 16, 2, 64, BF16)
    q, k, v = _fresh(1, 3, 4, 2, 64, BF16)
    mask, depths = _tree(1, 3)
    for args, error, match in (
            ((0,), ValueError, "at least"), ((2.5,), TypeError, "int"), ((9, mask), ValueError, "depths"), ((9, mask, depths.long()), TypeError, "int32"),
            ((9, mask, depths[:, :2]), ValueError, "depths"), ((9, mask, depths.cpu()), ValueError, "same device"), ((9, mask[:, :2], depths), ValueError, "mask"),
            ((9, None, [0, 1, 2]), TypeError, "int32")):
        with pytest.raises(error, match=match):
            window_tree_attention(q, k, v, *cache, *args)
    with pytest.raises(ValueError, match="at least"):
        window_tree_attention(q, k, v, *cache, 9, sinks=-1)
    with pytest.raises(RuntimeError, match="window_tree_attention has no gradient"):
        window_tree_attention(q.requires_grad_(True), k, v, *cache, 9)
