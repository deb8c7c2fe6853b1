"""GPU tests of accumulated weights where something is not finite or names no page: they follow from queries, keys and the page
table, and values do not enter them."""

from __future__ import annotations

import math

import pytest
import torch

from gdn2_sm120_b200.eviction import weighed_attention, weighed_attention_varlen, weighed_token_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _inputs(lead, heads, kv_heads, dim, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(*lead, h, dim, generator=gen, device=DEV).to(BF16) for h in (heads, kv_heads, kv_heads)]


def _cache(batch, cached, tokens, seed=0):
    page, kv_heads, dim = 16, 2, 64
    gen = torch.Generator(device=DEV).manual_seed(seed)
    columns = -(-(cached + tokens) // page)
    pages = [torch.randn(batch * columns + 2, page, kv_heads, dim, generator=gen, device=DEV).to(BF16) for _ in range(2)]
    weights = torch.rand(batch * columns + 2, kv_heads, page, generator=gen, device=DEV)
    table = torch.randperm(batch * columns, generator=gen, device=DEV).int().view(batch, columns)
    lengths = torch.full((batch,), cached, device=DEV, dtype=torch.int32)
    places = torch.arange(cached, cached + tokens, device=DEV).expand(batch, -1)
    return [*pages, weights, table, lengths], table.long().gather(1, places // page) * page + places % page


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_values_do_not_enter_the_weights_of_prompts(what):
    q, k, v = _inputs((1, 400), 4, 2, 64)
    want = weighed_attention(q, k, v)
    strange = v.clone()
    strange[0, 100:300, 1] = what
    out, weights = weighed_attention(q, k, strange)
    assert not torch.isfinite(out[0, 100:, 2:]).any() and torch.equal(weights, want[1])
    packed = weighed_attention_varlen(q, k, strange, (0, 250, 400))[1]
    assert torch.equal(packed, weighed_attention_varlen(q, k, v, (0, 250, 400))[1]) and torch.isfinite(packed).all()


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_values_do_not_enter_the_weights_of_steps(what):
    cache, slots = _cache(2, 300, 3)
    q, k, v = _inputs((2, 3), 4, 2, 64)
    clean = [x.clone() for x in cache]
    weighed_token_attention(q, k, v, *clean, slots)
    cache[1][cache[3][0, 4].long(), 3] = what
    v[1, 0] = what
    out = weighed_token_attention(q, k, v, *cache, slots)
    assert not torch.isfinite(out).any() and torch.equal(cache[2], clean[2]) and torch.isfinite(cache[2]).all()


@pytest.mark.parametrize("bad", [-1, 10 ** 9])
@pytest.mark.parametrize("tokens,decay", [(1, 1.0), (3, 0.5), (40, 0.0)])
def test_a_page_number_outside_the_cache_makes_its_sequences_weights_nan(tokens, decay, bad):
    """Those of its tokens in good pages and of its new ones; the others' and all other places keep their bits."""

    cache, slots = _cache(3, 300, tokens, seed=tokens)
    q, k, v = _inputs((3, tokens), 4, 2, 64)
    table = cache[3].clone()
    clean = [x.clone() for x in cache]
    weighed_token_attention(q, k, v, *clean, slots, decay=decay)
    before = cache[2].clone()
    cache[3][1, 5] = bad
    out = weighed_token_attention(q, k, v, *cache, slots, decay=decay)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()
    t = torch.arange(300 + tokens, device=DEV)
    touched = torch.zeros_like(before, dtype=torch.bool)
    for b in range(3):
        pages = table[b, t // 16].long()
        got, want = cache[2][pages, :, t % 16], clean[2][pages, :, t % 16]
        if b != 1:
            assert torch.equal(got, want)
        else:
            lost = t // 16 == 5         # what the page that has no number any more held
            assert torch.isnan(got[~lost]).all() and torch.equal(got[lost], before[pages, :, t % 16][lost])
        touched[pages, :, t % 16] = True
    assert torch.equal(cache[2][~touched], before[~touched])


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_scores_that_are_nan_or_infinite_make_weights_nan(what):
    """Those of the tokens that a query with such a score sees, in its key head, and no others."""

    q, k, v = _inputs((1, 300), 4, 2, 64)
    q[..., 0] = q[..., 0].abs() + 0.5
    want = weighed_attention(q, k, v)[1]
    strange = k.clone()
    strange[0, 299, 1, 0] = what          # the last query alone sees it
    weights = weighed_attention(q, strange, v)[1]
    assert torch.isnan(weights[0, :, 1]).all() and torch.equal(weights[0, :, 0], want[0, :, 0])
    cache, slots = _cache(2, 300, 3)
    q, k, v = _inputs((2, 3), 4, 2, 64)
    q[..., 0] = q[..., 0].abs() + 0.5
    clean = [x.clone() for x in cache]
    weighed_token_attention(q, k, v, *clean, slots)
    cache[0][cache[3][0, 4].long(), 3, 1, 0] = what
    weighed_token_attention(q, k, v, *cache, slots)
    places = torch.arange(303, device=DEV)
    for b in range(2):
        pages = cache[3][b, places // 16].long()
        got, kept = cache[2][pages, :, places % 16], clean[2][pages, :, places % 16]
        assert torch.equal(got[:, 0], kept[:, 0])
        assert torch.isnan(got[:, 1]).all() if b == 0 else torch.equal(got[:, 1], kept[:, 1])
