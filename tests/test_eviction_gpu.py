"""GPU tests of accumulated attention weights and of eviction by them, against plain forms in 64 bits.

Weights are sums of exponentials of scores in 32 bits, never rounded to fewer: what attention_bounds allows for all that is in 32 bits,
2^-13 of the sum (its terms are positive), is what a weight may be off by, and half a spacing of 32-bit floats below their normal
range for every term."""

from __future__ import annotations

import math

import pytest
import torch

import attention_bounds as exact
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen
from gdn2_sm120_b200.eviction import evict_tokens, weighed_attention, weighed_attention_varlen, weighed_token_attention
from gdn2_sm120_b200.paged import append_tokens, tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _normal(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _inputs(lead, heads, kv_heads, dim, dtype, seed=0):
    return [_normal(*lead, h, dim, dtype=dtype, seed=seed + i) for i, h in enumerate((heads, kv_heads, kv_heads))]


def _softmax(q, k, seen, scale):
    """[H, N, M] in 64 bits; rows that see nothing are 0"""

    group = q.shape[1] // k.shape[1]
    q, k = q.double().transpose(0, 1), k.double().transpose(0, 1).repeat_interleave(group, 0)
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    return torch.softmax(s, -1).nan_to_num(0.0)


def _received(q, k, seen, scale):
    p = _softmax(q, k, seen, scale).sum(1)
    return p.view(k.shape[1], -1, p.shape[1]).sum(1).T     # [M, Hkv]


def _close(got, want, terms, what=""):
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).abs()
    allowed = 2.0 ** -13 * want + terms * 2.0 ** -126
    assert (off <= allowed).all(), f"{what}: {(off / allowed.clamp_min(1e-300)).max().item():.3f} times its bound"


# ---- prompts -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("batch,time,heads,kv_heads,dim", [
    (1, 1, 1, 1, 128), (2, 2, 2, 1, 64), (3, 63, 4, 2, 128), (1, 64, 2, 2, 8), (2, 65, 6, 2, 40), (1, 127, 3, 1, 64), (2, 128, 2, 1, 128),
    (1, 129, 4, 4, 72), (1, 255, 2, 2, 128), (2, 256, 2, 1, 96), (1, 257, 8, 1, 128), (2, 511, 2, 2, 64), (1, 777, 3, 3, 120), (1, 1500, 16, 1, 128),
    (40, 300, 8, 4, 64),
])
def test_weights_of_a_batch(dtype, batch, time, heads, kv_heads, dim):
    q, k, v = _inputs((batch, time), heads, kv_heads, dim, dtype, seed=time)
    out, weights = weighed_attention(q, k, v)
    assert torch.equal(out, causal_attention(q, k, v))
    assert weights.shape == (batch, time, kv_heads) and weights.dtype == FP32 and weights.is_contiguous()
    for b in range(min(batch, 4)):
        _close(weights[b], _received(q[b], k[b], exact.causal(time, DEV), dim ** -0.5), time * heads, f"sequence {b}")
    total = weights.double().sum((1, 2))        # every query gives away 1
    assert ((total - time * heads).abs() <= 2.0 ** -13 * time * heads).all()
    assert torch.equal(weights, weighed_attention(q, k, v)[1])


@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [
    ((1,), 1, 1, 64), ((0, 5, 0, 0, 130, 1, 0), 4, 2, 128), ((128, 256, 64, 1, 1, 383), 2, 1, 64), ((1000, 3, 500), 3, 3, 96),
    ((2000, 30, 1, 700), 16, 1, 128), (tuple((7 * i) % 61 for i in range(600)), 2, 1, 64),
])
def test_weights_of_packed_sequences(lengths, heads, kv_heads, dim):
    bounds = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    q, k, v = _inputs((1, bounds[-1]), heads, kv_heads, dim, BF16, seed=3)
    out, weights = weighed_attention_varlen(q, k, v, bounds)
    assert torch.equal(out, causal_attention_varlen(q, k, v, bounds))
    for lo, hi in list(zip(bounds, bounds[1:]))[::max(1, len(lengths) // 20)]:
        if hi > lo:
            want = _received(q[0, lo:hi], k[0, lo:hi], exact.causal(hi - lo, DEV), dim ** -0.5)
            _close(weights[0, lo:hi], want, (hi - lo) * heads, f"rows {lo} to {hi}")
    assert torch.equal(weights, weighed_attention_varlen(q, k, v, torch.tensor(bounds))[1])


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_weights_with_other_scales_and_of_views(scale):
    fused = _normal(2, 300, 8, 64, dtype=BF16, seed=1)
    q, k, v = fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:]
    out, weights = weighed_attention(q, k, v, scale=scale)
    assert torch.equal(out, causal_attention(q, k, v, scale=scale))
    for b in range(2):
        _close(weights[b], _received(q[b], k[b], exact.causal(300, DEV), scale), 1200)


@pytest.mark.parametrize("height", [60.0, 400.0, 100000.0])
def test_weights_where_scores_are_far_apart(height):
    """Single scores far above all others, near and far references: their columns get all of what comes behind them."""

    time, dim = 520, 64
    q, k, v = _inputs((1, time), 2, 1, dim, BF16, seed=11)
    q[..., 1:], k[..., 1:] = 0.0, 0.0
    q[..., 0], k[..., 0] = 4.0, 0.0
    for at, share in ((3, 0.25), (140, 0.5), (300, 0.75), (511, 1.0)):
        k[0, at, 0, 0] = height * share / 4.0
    _, weights = weighed_attention(q, k, v, scale=1.0)
    _close(weights[0], _received(q[0], k[0], exact.causal(time, DEV), 1.0), 2 * time)


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_weights_of_packed_sequences_do_not_meet(what):
    bounds = (0, 100, 265, 400)
    q, k, v = _inputs((1, 400), 4, 2, 64, BF16, seed=4)
    want = weighed_attention_varlen(q, k, v, bounds)
    for lo, hi in ((0, 100), (265, 400)):
        inputs = [x.clone() for x in (q, k, v)]
        for x in inputs:
            x[:, lo:hi] = what
        got = weighed_attention_varlen(*inputs, bounds)
        _close(got[1][0, 100:265], _received(q[0, 100:265], k[0, 100:265], exact.causal(165, DEV), 64 ** -0.5), 660)
        assert torch.isnan(got[1][0, lo]).all() and (not math.isnan(what) or torch.equal(got[1][0, 100:265], want[1][0, 100:265]))


def test_a_query_that_is_nan_makes_the_weights_of_what_it_sees_nan():
    q, k, v = _inputs((1, 400), 4, 2, 64, BF16, seed=5)
    q[0, 200, 3, 7] = math.nan
    _, weights = weighed_attention(q, k, v)
    clean = q.clone()
    clean[0, 200, 3] = 0.0
    want = weighed_attention(clean, k, v)[1]
    assert torch.isnan(weights[0, :201, 1]).all()
    assert torch.equal(weights[0, 201:], want[0, 201:]) and torch.equal(weights[0, :, 0], want[0, :, 0])


def test_weights_on_another_stream_and_in_a_graph():
    q, k, v = _inputs((2, 300), 8, 2, 64, BF16, seed=6)
    want = weighed_attention(q, k, v)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = weighed_attention(q, k, v)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = weighed_attention(q, k, v)
    q.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(weighed_attention(q, k, v), got))


def test_weights_of_no_tokens_and_refusals():
    q, k, v = _inputs((2, 0), 4, 2, 64, BF16)
    out, weights = weighed_attention(q, k, v)
    assert out.shape == q.shape and weights.shape == (2, 0, 2)
    q, k, v = _inputs((1, 8), 4, 2, 64, BF16)
    with pytest.raises(TypeError, match="dtype"):
        weighed_attention(q, k.half(), v)
    with pytest.raises(ValueError, match="scale"):
        weighed_attention(q, k, v, scale=math.nan)
    with pytest.raises(ValueError):
        weighed_attention_varlen(q, k, v, (0, 9))
    with pytest.raises(RuntimeError, match="no gradient"):
        weighed_attention(q.requires_grad_(True), k, v)
    with torch.no_grad():
        assert torch.equal(weighed_attention(q, k, v)[0], causal_attention(q, k, v))


# ---- new tokens over a cache -----------------------------------------------------------------------------------------


def _cache(lengths, room, page, kv_heads, dim, dtype, seed=0, fill=None):
    """Pages in no order with `room` places behind every sequence: pages, weights, table, lengths and the new tokens' slots."""

    gen = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-(n + room) // page) for n in lengths]
    pages = sum(need) + 3
    k, v = (torch.randn(pages, page, kv_heads, dim, generator=gen, device=DEV).to(dtype) for _ in range(2))
    weights = torch.rand(pages, kv_heads, page, generator=gen, device=DEV)
    order = torch.randperm(pages, generator=gen, device=DEV).int()
    table = torch.full((len(lengths), max(need)), -5, device=DEV, dtype=torch.int32)
    slots, at = [], 0
    for b, (n, count) in enumerate(zip(lengths, need)):
        table[b, :count] = order[at:at + count]
        at += count
        t = torch.arange(n, n + room, device=DEV)
        slots.append(table[b, t // page].long() * page + t % page)
        if fill is not None and n % page:
            k[table[b, n // page].long(), n % page:], v[table[b, n // page].long(), n % page:] = fill, fill
    return [k, v, weights, table, torch.tensor(lengths, device=DEV, dtype=torch.int32)], torch.stack(slots)


def _check_step(out, weights, before, q, k, v, cache, slots, decay, scale=None):
    k_pages, v_pages, _, table, lengths = cache
    page, tokens, dim = k_pages.shape[1], q.shape[1], q.shape[3]
    scale = dim ** -0.5 if scale is None else scale
    touched = torch.zeros_like(weights, dtype=torch.bool)
    for b in range(q.shape[0]):
        n = int(lengths[b])
        t = torch.arange(n, device=DEV)
        pages = table[b, t // page].long()
        keys, values = (torch.cat([x[pages, t % page], y[b]]) for x, y in ((k_pages, k), (v_pages, v)))
        seen = torch.cat([torch.ones(tokens, n, device=DEV, dtype=torch.bool), exact.causal(tokens, DEV)], 1)
        want = exact.attention(*(x.transpose(0, 1) for x in (q[b], keys, values)), seen, scale)
        exact.check(f"sequence {b}", out[b], *want["o"])
        got = _received(q[b], keys, seen, scale)
        old = before[pages, :, t % page].double() * decay if decay else 0.0
        rows = q.shape[1] * q.shape[2]
        _close(weights[pages, :, t % page], old + got[:n], rows + 1, f"cached weights {b}")
        touched[pages, :, t % page] = True
        new = slots[b] >= 0
        _close(weights[slots[b][new] // page, :, slots[b][new] % page], got[n:][new], rows, f"new weights {b}")
        touched[slots[b][new] // page, :, slots[b][new] % page] = True
    assert torch.equal(weights[~touched], before[~touched])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,page,tokens,heads,kv_heads,dim,decay", [
    ((0,), 16, 1, 1, 1, 128, 1.0), ((1, 0, 15, 16, 17), 16, 1, 4, 1, 64, 0.5), ((63, 64, 65), 64, 1, 8, 8, 128, 1.0),
    ((500, 3), 24, 2, 6, 2, 96, 0.0), ((129, 1000), 7, 1, 16, 1, 128, 1.0), ((300,), 128, 1, 17, 1, 128, 1.0), ((40, 260, 0), 16, 16, 2, 1, 8, 0.25),
    ((64, 128, 777), 32, 5, 32, 4, 72, 1.0), ((200, 90), 1, 3, 64, 1, 64, 0.0), ((70, 2000), 16, 64, 8, 2, 128, 1.0), ((3000,) * 7, 64, 1, 4, 2, 64, 1.0),
])
def test_new_tokens_over_a_cache(dtype, lengths, page, tokens, heads, kv_heads, dim, decay):
    cache, slots = _cache(lengths, tokens, page, kv_heads, dim, dtype, fill=math.nan)
    if decay == 0.0:
        cache[2].fill_(math.nan)     # what is not read may be anything
    q, k, v = _inputs((len(lengths), tokens), heads, kv_heads, dim, dtype, seed=1)
    before = cache[2].clone()
    out = weighed_token_attention(q, k, v, *cache, slots, decay=decay)
    if decay == 0.0:
        before.nan_to_num_(0.0)
        cache[2].nan_to_num_(0.0)
    _check_step(out, cache[2], before, q, k, v, cache, slots, decay)
    if tokens * heads // kv_heads <= 16:
        assert torch.equal(out, tree_attention(q, k, v, *cache[:2], *cache[3:]))


def test_many_sequences_and_a_long_one():
    lengths = [(37 * i) % 200 for i in range(300)] + [30011]
    cache, slots = _cache(lengths, 1, 16, 1, 64, BF16)
    q, k, v = _inputs((301, 1), 2, 1, 64, BF16, seed=1)
    slots[5], slots[6], slots[300] = -1, cache[0].shape[0] * 16, 2 ** 62
    before = cache[2].clone()
    out = weighed_token_attention(q, k, v, *cache, slots)
    slots[6], slots[300] = -1, -1
    _check_step(out, cache[2], before, q, k, v, cache, slots, 1.0)


@pytest.mark.parametrize("height", [30.0, 400.0, 100000.0])
def test_steps_where_scores_are_far_apart(height):
    cache, slots = _cache((900,), 2, 16, 2, 64, BF16)
    q, k, v = _inputs((1, 2), 4, 2, 64, BF16, seed=1)
    for x in (q, k, cache[0]):
        x.zero_()
    q[..., 0] = 4.0
    for at, share in ((100, 0.25), (200, 0.4), (513, 0.6), (890, 1.0)):
        cache[0][cache[3][0, at // 16].long(), at % 16, :, 0] = height * share / 4.0
    before = cache[2].clone()
    out = weighed_token_attention(q, k, v, *cache, slots, scale=1.0)
    _check_step(out, cache[2], before, q, k, v, cache, slots, 1.0, 1.0)


def test_decoding_accumulates_what_one_prompt_gives():
    time, page, first = 150, 16, 40
    q, k, v = _inputs((1, time), 4, 2, 64, BF16, seed=2)
    table = torch.randperm(10, device=DEV).int()[None]
    place = torch.arange(time, device=DEV)
    slots = (table[0, place // page].long() * page + place % page)[None]
    pages = [torch.zeros(10, page, 2, 64, device=DEV, dtype=BF16) for _ in range(2)]
    weights = torch.full((10, 2, page), math.nan, device=DEV)
    _, prompt = weighed_attention(q[:, :first], k[:, :first], v[:, :first])
    weights[slots[0, :first] // page, :, slots[0, :first] % page] = prompt[0]
    append_tokens(k[:, :first], v[:, :first], *pages, slots[:, :first])
    for at in range(first, time):
        now = slice(at, at + 1)
        length = torch.tensor([at], device=DEV, dtype=torch.int32)
        weighed_token_attention(q[:, now], k[:, now], v[:, now], *pages, weights, table, length, slots[:, now])
        append_tokens(k[:, now], v[:, now], *pages, slots[:, now])
    want = _received(q[0], k[0], exact.causal(time, DEV), 64 ** -0.5)
    _close(weights[slots[0] // page, :, slots[0] % page], want, time * 4)


def test_bad_pages_and_lengths():
    for tokens in (1, 3):
        cache, slots = _cache((300, 300, 300, 300), tokens, 16, 2, 64, BF16)
        q, k, v = _inputs((4, tokens), 4, 2, 64, BF16, seed=3)
        clean = [x.clone() for x in cache]
        want = weighed_token_attention(q, k, v, *clean, slots)
        before = cache[2].clone()
        cache[3][1, 5] = cache[0].shape[0]
        cache[4][2], cache[4][3] = -1, cache[3].shape[1] * 16 + 1
        out = weighed_token_attention(q, k, v, *cache, slots)
        assert torch.equal(out[0], want[0]) and torch.isnan(out[1:]).all()
        row = cache[3][0].long()
        assert torch.equal(cache[2][row], clean[2][row])
        for b in (2, 3):     # cached weights stay, new ones are NaN
            left = torch.ones(300 + tokens, device=DEV, dtype=torch.bool)
            t = torch.arange(300 + tokens, device=DEV)
            got = cache[2][clean[3][b, t // 16].long(), :, t % 16]
            assert torch.equal(got[:300], before[clean[3][b, t // 16].long(), :, t % 16][:300]) and torch.isnan(got[300:]).all() and left.all()


def test_a_captured_step_two_graphs_and_another_stream():
    cache, slots = _cache((900, 500), 1, 16, 2, 64, BF16)
    q, k, v = _inputs((2, 1), 8, 2, 64, BF16, seed=4)
    others = [x.clone() for x in cache]
    weighed_token_attention(q, k, v, *[x.clone() for x in cache], slots)
    graphs = []
    for c in (cache, others):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, weighed_token_attention(q, k, v, *c, slots, decay=0.5), c))
    want = [x.clone() for x in cache]
    for length in (900, 77, 0):
        cache[4][0] = others[4][0] = want[4][0] = length
        result = weighed_token_attention(q, k, v, *want, slots, decay=0.5)
        for graph, out, c in graphs:
            graph.replay()
        for graph, out, c in graphs:
            assert torch.equal(out, result) and torch.equal(c[2], want[2])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = weighed_token_attention(q, k, v, *others, slots, decay=0.5)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out, weighed_token_attention(q, k, v, *want, slots, decay=0.5)) and torch.equal(others[2], want[2])


def test_refusals_of_steps():
    cache, slots = _cache((40,), 1, 16, 2, 64, BF16)
    q, k, v = _inputs((1, 1), 4, 2, 64, BF16)
    k_pages, v_pages, weights, table, lengths = cache
    for args, error, match in (
            ((k_pages, v_pages, weights.half(), table, lengths, slots), TypeError, "float32"),
            ((k_pages, v_pages, weights.transpose(1, 2).contiguous(), table, lengths, slots), ValueError, "weight_pages"),
            ((k_pages, v_pages, None, table, lengths, slots), TypeError, "weight_pages"),
            ((k_pages, v_pages, weights.cpu(), table, lengths, slots), ValueError, "same device"),
            ((k_pages, v_pages, weights, table.long(), lengths, slots), TypeError, "int32"),
            ((k_pages, v_pages, weights, table, lengths, slots.int()), TypeError, "int64"),
            ((k_pages, v_pages, weights, table, lengths, slots[0]), ValueError, "slots"),
            ((k_pages, v_pages[:2], weights, table, lengths, slots), ValueError, "same shape"),
            ((k_pages, v_pages, lengths.new_zeros(0).float().new_empty(0), table, lengths, slots), ValueError, "weight_pages")):
        with pytest.raises(error, match=match):
            weighed_token_attention(q, k, v, *args)
    for decay in (-0.1, 1.5, math.nan, None, "1"):
        with pytest.raises(ValueError, match="decay"):
            weighed_token_attention(q, k, v, *cache, slots, decay=decay)
    with pytest.raises(NotImplementedError, match="256"):
        weighed_token_attention(*_inputs((1, 129), 4, 2, 64, BF16), *cache, slots.expand(1, 129).contiguous())
    with pytest.raises(RuntimeError, match="no gradient"):
        weighed_token_attention(q.clone().requires_grad_(True), k, v, *cache, slots)
    empty = _inputs((1, 0), 4, 2, 64, BF16)
    assert weighed_token_attention(*empty, *cache, slots[:, :0]).shape == empty[0].shape


# ---- eviction ----------------------------------------------------------------------------------------------------------


def _order(weights):
    """Numbers in the order that eviction goes by, in 64 bits: NaN above infinity, which is below what has to stay."""

    return torch.where(weights.isnan(), 1e305, weights.double().clamp(-1e300, 1e300))


def _check_eviction(before, after, table, lengths, new_table, new_lengths, keep, sinks, recent):
    (k0, v0, w0), (k1, v1, w1) = ([x.cpu() for x in y] for y in (before, after))
    pages, page, kv_heads, _ = k0.shape
    written = torch.zeros(pages, kv_heads, page, dtype=torch.bool)
    for b, n in enumerate(lengths.tolist()):
        assert int(new_lengths[b]) == min(n, keep)
        t = torch.arange(n)
        source, place = table[b].cpu().long()[t // page], t % page
        for head in range(kv_heads):
            if n <= keep:
                kept = t
            else:
                w = _order(w0[source, head, place])
                w[:sinks], w[n - recent:] = math.inf, math.inf
                kept = w.sort(descending=True, stable=True).indices[:keep].sort().values
            j = torch.arange(len(kept))
            to, at = new_table[b].cpu().long()[j // page], j % page
            there = (to >= 0) & (to < pages)
            kept, to, at = kept[there], to[there], at[there]
            written[to, head, at] = True
            for x, y in ((k0, k1), (v0, v1)):
                assert torch.equal(y[to, at, head], x[source[kept], place[kept], head])
            assert torch.equal(w1[to, head, at].nan_to_num(7.0), w0[source[kept], head, place[kept]].nan_to_num(7.0))
    untouched = ~written
    assert torch.equal(w1[untouched].nan_to_num(7.0), w0[untouched].nan_to_num(7.0))
    for x, y in ((k0, k1), (v0, v1)):
        assert torch.equal(y.transpose(1, 2)[untouched], x.transpose(1, 2)[untouched])


def _evicting(lengths, page, kv_heads, dim, keep, dtype=BF16, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    need, new = [-(-n // page) for n in lengths], -(-keep // page)
    pages = sum(need) + new * len(lengths) + 2
    k, v = (torch.randn(pages, page, kv_heads, dim, generator=gen, device=DEV).to(dtype) for _ in range(2))
    weights = torch.empty(pages, kv_heads, page, device=DEV).exponential_(1.0, generator=gen)
    order = torch.randperm(pages, generator=gen, device=DEV).int()
    table = torch.full((len(lengths), max(1, *need)), -5, device=DEV, dtype=torch.int32)
    at = 0
    for b, count in enumerate(need):
        table[b, :count] = order[at:at + count]
        at += count
    new_table = order[at:at + new * len(lengths)].view(len(lengths), new).clone()
    return [k, v, weights], table, torch.tensor(lengths, device=DEV, dtype=torch.int32), new_table


def _evict(cache, table, lengths, new_table, keep, sinks, recent):
    before = [x.clone() for x in cache]
    new_lengths = evict_tokens(*cache, table, lengths, new_table, keep, sinks=sinks, recent=recent)
    _check_eviction(before, cache, table, lengths, new_table, new_lengths, keep, sinks, recent)
    assert new_lengths.dtype == torch.int32


@pytest.mark.parametrize("lengths,page,kv_heads,dim,keep,sinks,recent,dtype", [
    ((1,), 16, 1, 64, 1, 0, 0, BF16), ((2,), 16, 1, 64, 1, 0, 0, FP16), ((5, 0, 3), 1, 2, 8, 3, 1, 1, BF16), ((100, 33, 0, 32, 31), 16, 2, 64, 32, 4, 8, FP16),
    ((513, 512, 511), 64, 3, 128, 200, 0, 200, BF16), ((700, 300), 24, 1, 96, 256, 100, 100, FP32), ((1000,), 7, 2, 40, 999, 1, 0, BF16),
    ((2100, 2049, 64), 128, 4, 128, 2048, 4, 64, BF16), ((5000, 4097), 16, 2, 64, 1, 0, 0, FP16), ((5000, 4097), 16, 2, 64, 1, 1, 0, BF16),
    ((3000,), 32, 1, 5, 1234, 7, 77, FP32), ((3000,), 32, 1, 3, 1234, 7, 77, BF16), ((777,), 48, 2, 2, 600, 3, 0, FP16), ((60000, 100), 64, 1, 8, 9000, 4, 1000, BF16),
])
def test_eviction(lengths, page, kv_heads, dim, keep, sinks, recent, dtype):
    _evict(*_evicting(lengths, page, kv_heads, dim, keep, dtype), keep, sinks, recent)


@pytest.mark.parametrize("kind", ["zeros", "same", "two", "few", "negative", "special", "tiny", "rising", "falling", "spread"])
def test_eviction_by_weights_of_any_kind(kind):
    """Many equal ones, of which the earlier stay; both zeros are equal; infinities, NaN and subnormal numbers."""

    for keep, sinks, recent in ((400, 0, 0), (400, 3, 50), (1, 0, 0), (1499, 0, 1)):
        cache, table, lengths, new_table = _evicting((1500, 700), 16, 2, 16, keep, seed=keep)
        w = cache[2]
        gen = torch.Generator(device=DEV).manual_seed(1)
        if kind == "zeros":
            w.copy_(torch.where(torch.rand(w.shape, generator=gen, device=DEV) < 0.5, 0.0, -0.0))
        elif kind == "same":
            w.fill_(0.7)
        elif kind == "two":
            w.copy_((w > 0.7).float())
        elif kind == "few":
            w.copy_((w * 3).round())
        elif kind == "negative":
            w.sub_(1.0)
        elif kind == "special":
            pick = torch.randint(0, 9, w.shape, generator=gen, device=DEV)
            for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0)):
                w[pick == i] = x
        elif kind == "tiny":
            w.mul_(1e-42)
        elif kind == "spread":
            w.copy_(10.0 ** (76 * torch.rand(w.shape, generator=gen, device=DEV) - 38))
        else:
            t = torch.arange(table.shape[1] * 16, device=DEV).float() * (1 if kind == "rising" else -1)
            for b, n in enumerate((1500, 700)):
                columns = -(-n // 16)
                w[table[b, :columns].long()] = t[:columns * 16].view(columns, 1, 16).expand(-1, 2, -1)
        _evict(cache, table, lengths, new_table, keep, sinks, recent)


def test_sequences_that_are_passed_by_and_shared_pages():
    cache, table, lengths, new_table = _evicting((500, 300, 400), 16, 2, 64, 128)
    new_table[1] = -1
    new_table[2, 3:] = cache[0].shape[0]
    table[2, :10] = table[0, :10]        # a common beginning
    _evict(cache, table, lengths, new_table, 128, 4, 20)


def test_bad_pages_and_lengths_evict_nothing():
    cache, table, lengths, new_table = _evicting((500, 500, 500, 500, 100), 16, 2, 64, 128)
    before = [x.clone() for x in cache]
    table[1, 30], table[4, 2] = -1, cache[0].shape[0]
    lengths[2], lengths[3] = -1, table.shape[1] * 16 + 1
    new_lengths = evict_tokens(*cache, table, lengths, new_table, 128)
    assert new_lengths.tolist() == [128, -1, -1, -1, -1]
    others = torch.ones(cache[0].shape[0], device=DEV, dtype=torch.bool)
    others[new_table[0].long()] = False
    assert all(torch.equal(a[others], b[others]) for a, b in zip(cache, before))
    assert not torch.equal(cache[0][new_table[0].long()], before[0][new_table[0].long()])


def test_more_weights_than_fit_into_shared_memory():
    cache, table, lengths, new_table = _evicting((70001, 50000), 128, 1, 8, 3000)
    cache[2].copy_((cache[2] * 50).round() / 50)      # many equal ones
    _evict(cache, table, lengths, new_table, 3000, 5, 100)


def test_a_captured_eviction():
    cache, table, lengths, new_table = _evicting((900, 500), 16, 2, 64, 256)
    start = [x.clone() for x in cache]
    evict_tokens(*[x.clone() for x in cache], table, lengths, new_table, 256, sinks=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new_lengths = evict_tokens(*cache, table, lengths, new_table, 256, sinks=2)
    for first, second in ((900, 500), (400, 20), (257, 256)):
        lengths.copy_(torch.tensor([first, second]))
        for x, y in zip(cache, start):
            x.copy_(y)
        start[2].copy_(start[2].flip(0))
        cache[2].copy_(start[2])
        graph.replay()
        _check_eviction(start, cache, table, lengths, new_table, new_lengths, 256, 2, 0)


def test_refusals_of_evictions():
    cache, table, lengths, new_table = _evicting((100,), 16, 2, 64, 32)
    for keep, sinks, recent, error in ((0, 0, 0, ValueError), (32, 20, 13, ValueError), (32, -1, 0, ValueError), (32, 0, -1, ValueError),
                                       (33, 0, 0, ValueError), (2.0, 0, 0, TypeError), (None, 0, 0, TypeError), (True, 0, 0, TypeError)):
        with pytest.raises(error):
            evict_tokens(*cache, table, lengths, new_table, keep, sinks=sinks, recent=recent)
    for args, error, match in (
            ((cache[0].long(), *cache[1:], table, lengths, new_table), TypeError, "bfloat16"),
            ((cache[0], cache[1].half(), cache[2], table, lengths, new_table), TypeError, "dtype"),
            ((cache[0], cache[0], cache[2], table, lengths, new_table), ValueError, "overlap"),
            ((*cache[:2], cache[2].double(), table, lengths, new_table), TypeError, "float32"),
            ((*cache[:2], cache[0].view(torch.float32).view(-1)[:cache[2].numel()].view(cache[2].shape), table, lengths, new_table), ValueError, "overlap"),
            ((*cache, table.long(), lengths, new_table), TypeError, "int32"), ((*cache, table, lengths.long(), new_table), TypeError, "int32"),
            ((*cache, table, lengths, new_table.long()), TypeError, "int32"), ((*cache, table, lengths[:0], new_table), ValueError, ""),
            ((*cache, table, lengths, new_table[:, :1]), ValueError, "room")):
        with pytest.raises(error, match=match):
            evict_tokens(*args, 32)
