"""GPU tests of the paged cache: writing tokens, and attention of drafted tokens over it, against plain attention in 64
bits within bounds that follow from what the kernels round (tests/attention_bounds.py)."""

from __future__ import annotations

import math

import pytest
import torch

import attention_bounds as exact
from gdn2_sm120_b200.attention import causal_attention
from gdn2_sm120_b200.paged import append_tokens, tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _cache(lengths, page, kv_heads, dim, dtype, seed=0, fill=None, spare=3):
    """Pages in no order; places that no sequence has hold `fill` (or noise)."""

    gen = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages, columns = sum(need) + spare, max(1, *need)
    k, v = (torch.randn(pages, page, kv_heads, dim, generator=gen, device=DEV).to(dtype) for _ in range(2))
    order = torch.randperm(pages, generator=gen, device=DEV).int()
    table = torch.full((len(lengths), columns), -5, device=DEV, dtype=torch.int32)   # unused entries name no page
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    if fill is not None:
        used = torch.zeros(pages, page, device=DEV, dtype=torch.bool)
        for i, n in enumerate(lengths):
            t = torch.arange(n, device=DEV)
            used[table[i, t // page].long(), t % page] = True
        k[~used], v[~used] = fill, fill
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
    return mask


def _check(out, q, k, v, cache, mask, scale=None):
    k_pages, v_pages, table, lengths = cache
    page, drafted, dim = k_pages.shape[1], q.shape[1], q.shape[3]
    for b in range(q.shape[0]):
        n = int(lengths[b])
        t = torch.arange(n, device=DEV)
        keys, values = (torch.cat([x[table[b, t // page].long(), t % page], y[b]]) for x, y in ((k_pages, k), (v_pages, v)))
        tail = mask if mask.ndim == 2 else mask[b]
        seen = torch.cat([torch.ones(drafted, n, device=DEV, dtype=torch.bool), tail], 1)
        want = exact.attention(*(x.transpose(0, 1) for x in (q[b], keys, values)), seen, scale or dim ** -0.5)
        exact.check(f"sequence {b}", out[b], *want["o"])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,page,drafted,heads,kv_heads,dim", [
    ((0,), 16, 1, 1, 1, 128), ((1, 0, 15, 16, 17), 16, 1, 4, 1, 64), ((63, 64, 65), 64, 1, 8, 8, 128),
    ((500, 3), 24, 2, 6, 2, 96), ((129, 1000), 7, 5, 8, 2, 128), ((300,), 128, 7, 16, 2, 128),
    ((40, 260, 0), 16, 16, 2, 1, 8), ((64, 128, 777), 32, 33, 4, 2, 72), ((200, 90), 1, 48, 8, 1, 64),
    ((70,), 16, 64, 2, 2, 128), ((5, 400), 16, 65, 3, 1, 128), ((100,), 48, 130, 2, 1, 40),
])
def test_trees_over_a_cache(dtype, lengths, page, drafted, heads, kv_heads, dim):
    cache = _cache(lengths, page, kv_heads, dim, dtype, fill=math.nan)
    q, k, v = _fresh(len(lengths), drafted, heads, kv_heads, dim, dtype)
    mask = _tree(len(lengths), drafted)
    out = tree_attention(q, k, v, *cache, mask)
    assert out.shape == q.shape and out.is_contiguous()
    _check(out, q, k, v, cache, mask)
    chain = torch.ones(drafted, drafted, device=DEV, dtype=torch.bool).tril()
    plain = tree_attention(q, k, v, *cache)
    _check(plain, q, k, v, cache, chain)
    assert torch.equal(plain, tree_attention(q, k, v, *cache, chain))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("drafted,heads", [(2, 4), (20, 4), (40, 16)])
@pytest.mark.parametrize("height", [20.0, 400.0])
def test_single_scores_far_above_all_others(dtype, drafted, heads, height):
    """In the cache and among the drafts, in tiles of either chain: 4, 40 and 320 rows of a key head."""

    cache = _cache((900,), 16, 2, 64, dtype)
    q, k, v = _fresh(1, drafted, heads, 2, 64, dtype)
    q[..., 0], k[..., 0] = 4.0, 0.0
    cache[0][..., 0] = 0.0
    for at, share in ((100, 0.25), (200, 0.4), (513, 0.6), (890, 0.8)):
        cache[0][cache[2][0, at // 16].long(), at % 16, :, 0] = height * share / 4.0
    k[:, drafted - 1, :, 0] = height / 4.0
    mask = _tree(1, drafted)
    _check(tree_attention(q, k, v, *cache, mask, scale=1.0), q, k, v, cache, mask, 1.0)


def test_many_sequences_and_a_long_one():
    lengths = [(37 * i) % 200 for i in range(300)] + [30011]
    cache = _cache(lengths, 16, 1, 64, BF16)
    q, k, v = _fresh(301, 1, 2, 1, 64, BF16)
    _check(tree_attention(q, k, v, *cache), q, k, v, cache, torch.ones(1, 1, device=DEV, dtype=torch.bool))


def test_a_chain_over_an_empty_cache_is_causal_attention():
    q, k, v = _fresh(2, 100, 4, 2, 128, FP16)
    cache = _cache((0, 0), 16, 2, 128, FP16)
    out = tree_attention(q, k, v, *cache)
    for b in range(2):
        want = exact.attention(*(x[b].transpose(0, 1) for x in (q, k, v)), exact.causal(100, DEV), 128 ** -0.5)
        exact.check("chain", out[b], *want["o"])
        exact.check("causal", causal_attention(q, k, v)[b], *want["o"])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows_that_see_nothing_give_zero(dtype):
    lengths = (0, 0, 70)
    cache = _cache(lengths, 16, 2, 64, dtype, fill=math.inf)
    q, k, v = _fresh(3, 6, 4, 2, 64, dtype)
    mask = torch.zeros(3, 6, 6, device=DEV, dtype=torch.bool)
    mask[0, 1, 4] = mask[2, 5, 0] = True
    out = tree_attention(q, k, v, *cache, mask)
    _check(out, q, k, v, cache, mask)
    assert not out[0, 0].any() and not out[1].any() and out[0, 1].any() and out[2, 0].any()


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf, "lowest"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_masked_drafts_may_hold_anything(what, dtype):
    """A drafted token that some rows do not see reaches those that do and no others."""

    what = torch.finfo(dtype).min if what == "lowest" else what
    cache = _cache((130,), 16, 2, 64, dtype)
    q, k, v = _fresh(1, 9, 4, 2, 64, dtype)
    mask = _tree(1, 9)
    mask[0, :, 5] = False
    mask[0, 7, 5] = True
    clean = tree_attention(q, k, v, *cache, mask)
    for tensors in ((k,), (v,), (k, v)):
        kept = [x.clone() for x in tensors]
        for x in tensors:
            x[0, 5] = what
        out = tree_attention(q, k, v, *cache, mask)
        others = [i for i in range(9) if i != 7]
        assert torch.equal(out[0, others], clean[0, others])
        if v is tensors[-1] and not math.isfinite(what):
            assert not torch.isfinite(out[0, 7]).any()
        for x, y in zip(tensors, kept):
            x.copy_(y)
    # one value alone
    v[0, 5, 1, 3] = what
    out = tree_attention(q, k, v, *cache, mask)
    if not math.isfinite(what):
        bad = ~torch.isfinite(out[0, 7])
        assert bad[2:, 3].all() and bad.sum() == 2


def test_an_infinite_value_in_the_cache_reaches_every_row():
    cache = _cache((130,), 16, 1, 64, BF16)
    q, k, v = _fresh(1, 3, 2, 1, 64, BF16)
    cache[1][cache[2][0, 2].long(), 5, 0, 7] = math.inf
    out = tree_attention(q, k, v, *cache)
    assert torch.isinf(out[..., 7]).all() and torch.isfinite(out[..., :7]).all() and torch.isfinite(out[..., 8:]).all()


def test_pages_and_lengths_that_cannot_be_make_nan():
    lengths = (40, 40, 40, 40)
    k_pages, v_pages, table, counts = _cache(lengths, 16, 2, 64, BF16)
    q, k, v = _fresh(4, 3, 4, 2, 64, BF16)
    clean = tree_attention(q, k, v, k_pages, v_pages, table, counts)
    table = table.clone()
    table[0, 1] = k_pages.shape[0]
    table[1, 2] = -1
    counts = torch.tensor([40, 40, 16 * table.shape[1] + 1, -1], device=DEV, dtype=torch.int32)
    out = tree_attention(q, k, v, k_pages, v_pages, table, counts)
    assert torch.isnan(out).all()
    counts = torch.tensor([16, 32, 40, 40], device=DEV, dtype=torch.int32)    # the bad pages are out of reach now
    out = tree_attention(q, k, v, k_pages, v_pages, table, counts)
    assert torch.isfinite(out).all() and torch.equal(out[2:], clean[2:])


def test_views_and_other_integer_strides():
    cache = _cache((90, 33), 16, 2, 64, BF16)
    q, k, v = _fresh(2, 4, 4, 2, 64, BF16)
    mask = _tree(2, 4)
    want = tree_attention(q, k, v, *cache, mask)
    fused = torch.cat([q, k, v], 2)
    table = torch.stack([cache[2], cache[2]], 2)[..., 0]
    got = tree_attention(fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:], cache[0], cache[1], table,
                         torch.stack([cache[3], cache[3]], 1)[:, 0], mask.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(got, want)
    wide = torch.cat([cache[2], cache[2]], 1)[:, :cache[2].shape[1]]
    assert torch.equal(tree_attention(q, k, v, cache[0], cache[1], wide, cache[3], mask), want)


def test_negative_and_zero_scale():
    cache = _cache((90,), 16, 1, 64, BF16)
    q, k, v = _fresh(1, 4, 2, 1, 64, BF16)
    mask = _tree(1, 4)
    for scale in (-0.3, 1e-30):
        _check(tree_attention(q, k, v, *cache, mask, scale=scale), q, k, v, cache, mask, scale)
    assert torch.isfinite(tree_attention(q, k, v, *cache, mask, scale=0.0)).all()


def test_a_graph_is_replayed_with_other_lengths_and_pages():
    cache = _cache((300, 20), 16, 2, 128, BF16)
    q, k, v = _fresh(2, 3, 8, 2, 128, BF16)
    tree_attention(q, k, v, *cache)
    table, lengths = cache[2].clone(), cache[3].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tree_attention(q, k, v, cache[0], cache[1], table, lengths)
    lengths.copy_(torch.tensor([17, 20]))
    table[0, :2] = table[0, 3:5].clone()
    graph.replay()
    now = (cache[0], cache[1], table, lengths)
    _check(out, q, k, v, now, torch.ones(3, 3, device=DEV, dtype=torch.bool).tril())


def test_another_stream_and_the_same_bits_every_time():
    cache = _cache((700, 20, 5000), 16, 2, 128, BF16)
    q, k, v = _fresh(3, 3, 8, 2, 128, BF16)
    want = tree_attention(q, k, v, *cache)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        outs = [tree_attention(q, k, v, *cache) for _ in range(20)]
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, want) for x in outs)


@pytest.mark.slow
def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements: appended to and read from at its end."""

    page, kv_heads, dim = 64, 8, 128
    pages = 2 ** 31 // (page * kv_heads * dim) + 9
    k_pages, v_pages = (torch.empty(pages, page, kv_heads, dim, device=DEV, dtype=BF16) for _ in range(2))
    q, k, v = _fresh(1, 130, 8, kv_heads, dim, BF16)
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], device=DEV, dtype=torch.int32)
    t = torch.arange(130, device=DEV)
    append_tokens(k, v, k_pages, v_pages, (table[0, t // page].long() * page + t % page)[None])
    cache = (k_pages, v_pages, table, torch.tensor([130], device=DEV, dtype=torch.int32))
    q, k, v = _fresh(1, 2, 8, kv_heads, dim, BF16, seed=9)
    _check(tree_attention(q, k, v, *cache), q, k, v, cache, torch.ones(2, 2, device=DEV, dtype=torch.bool).tril())


# ---- writing tokens ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP16, torch.float32])
@pytest.mark.parametrize("tokens,page,kv_heads,dim", [(1, 1, 1, 1), (5, 16, 2, 64), (333, 24, 3, 40), (1000, 7, 8, 128), (64, 64, 1, 3)])
def test_append(dtype, tokens, page, kv_heads, dim):
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    pages = tokens // page + 3
    k, v = (torch.randn(tokens, kv_heads, dim, generator=gen, device=DEV).to(dtype) for _ in range(2))
    k_pages, v_pages = (torch.randn(pages, page, kv_heads, dim, generator=gen, device=DEV).to(dtype) for _ in range(2))
    slots = torch.randperm(pages * page, generator=gen, device=DEV)[:tokens]
    skipped = torch.rand(tokens, generator=gen, device=DEV) < 0.2
    out_of_range = torch.tensor([-1, pages * page, -2 ** 40, 2 ** 62], device=DEV)
    slots[skipped] = out_of_range[torch.arange(tokens, device=DEV) % 4][skipped]
    want_k, want_v = k_pages.clone(), v_pages.clone()
    keep = ~skipped
    want_k.view(-1, kv_heads, dim)[slots[keep]] = k[keep]
    want_v.view(-1, kv_heads, dim)[slots[keep]] = v[keep]
    got = append_tokens(k, v, k_pages, v_pages, slots)
    assert got[0] is k_pages and got[1] is v_pages
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)


def test_append_of_views_and_batches():
    batch, time, kv_heads, dim, page = 2, 21, 2, 64, 16
    gen = torch.Generator(device=DEV).manual_seed(0)
    fused = torch.randn(batch, time, 2 * kv_heads * dim + 1, generator=gen, device=DEV).bfloat16()
    slots = torch.randperm(4 * page, generator=gen, device=DEV)[:batch * time].view(batch, time)
    for begin in (0, 1):    # aligned to 16 bytes or not
        k, v = (fused[..., begin + i * kv_heads * dim:begin + (i + 1) * kv_heads * dim].unflatten(-1, (kv_heads, dim)) for i in range(2))
        pages = [torch.zeros(4, page, kv_heads, dim, device=DEV, dtype=BF16) for _ in range(4)]
        append_tokens(k, v, *pages[:2], slots)
        append_tokens(k.contiguous(), v.contiguous(), *pages[2:], slots)
        assert torch.equal(pages[0], pages[2]) and torch.equal(pages[1], pages[3])
        assert torch.equal(pages[0].view(-1, kv_heads, dim)[slots], k)
        # slots in another order, tokens cut from the middle, channels that are not contiguous
        append_tokens(k[:, 3:9], v[:, 3:9], *pages[:2], slots[:, 3:9])
        assert torch.equal(pages[0], pages[2])
        append_tokens(k[0].transpose(1, 2).contiguous().transpose(1, 2), v[0], *pages[:2], slots[0])
        assert torch.equal(pages[0], pages[2]) and torch.equal(pages[1], pages[3])
    assert append_tokens(k[:, :0], v[:, :0], *pages[:2], slots[:, :0])[0] is pages[0]


# ---- refusals ----------------------------------------------------------------------------------------------


def _good():
    q, k, v = _fresh(2, 3, 4, 2, 64, BF16)
    k_pages, v_pages, table, lengths = _cache((20, 30), 16, 2, 64, BF16)
    return dict(q=q, k=k, v=v, k_pages=k_pages, v_pages=v_pages, page_table=table, lengths=lengths, mask=_tree(2, 3))


@pytest.mark.parametrize("name,change,error", [
    ("q", lambda x: x.float(), TypeError), ("q", lambda x: x[0], ValueError), ("q", lambda x: x[:, :, :3].contiguous(), ValueError),
    ("q", lambda x: x[..., :60], NotImplementedError), ("k", lambda x: x[:, :2], ValueError), ("v", lambda x: x.half(), TypeError),
    ("k", lambda x: x.cpu(), ValueError), ("k_pages", lambda x: x[..., :32], ValueError), ("k_pages", lambda x: x.half(), TypeError),
    ("v_pages", lambda x: x[:2], ValueError), ("v_pages", lambda x: x.transpose(0, 1), ValueError), ("k_pages", lambda x: x[:0], ValueError),
    ("v_pages", lambda x: x.cpu(), ValueError), ("page_table", lambda x: x.long(), TypeError), ("page_table", lambda x: x[:1], ValueError),
    ("page_table", lambda x: x[:, :0], ValueError), ("page_table", lambda x: x.cpu(), ValueError), ("lengths", lambda x: x.long(), TypeError),
    ("lengths", lambda x: x[:1], ValueError), ("lengths", lambda x: None, TypeError), ("mask", lambda x: x.int(), TypeError),
    ("mask", lambda x: x[:, :2], ValueError), ("mask", lambda x: x.cpu(), ValueError), ("q", lambda x: x.requires_grad_(True), RuntimeError),
])
def test_tree_refusals(name, change, error):
    args = _good()
    args[name] = change(args[name])
    with pytest.raises(error):
        tree_attention(**args)


def test_append_refusals():
    k, v = (torch.zeros(4, 2, 64, device=DEV, dtype=BF16) for _ in range(2))
    pages = [torch.zeros(3, 16, 2, 64, device=DEV, dtype=BF16) for _ in range(2)]
    slots = torch.arange(4, device=DEV)
    for args, error in (
        ((k, v[:3], *pages, slots), ValueError), ((k, v.half(), *pages, slots), TypeError), ((k, v, *pages, slots.int()), TypeError),
        ((k, v, *pages, slots[:3]), ValueError), ((k.cpu(), v.cpu(), *pages, slots), ValueError), ((k, v, pages[0], pages[0], slots), ValueError),
        ((pages[0][0, :4], v, *pages, slots), ValueError), ((k, v, pages[0][..., :32], pages[1], slots), ValueError),
        ((k, v, pages[0].transpose(0, 1), pages[1], slots), ValueError), ((k.int(), v.int(), *pages, slots), TypeError),
        ((k[0], v[0], *pages, slots), ValueError), ((None, v, *pages, slots), TypeError),
    ):
        with pytest.raises(error):
            append_tokens(*args)


@pytest.mark.parametrize("batched", [False, True])
def test_append_is_seen_by_autograd(batched):
    """A cache that a backward has saved and that is written to afterwards gives an error, and no wrong gradient."""

    k, v = (torch.randn(1, 4, 2, 64, device=DEV) for _ in range(2))
    slots = torch.arange(4, device=DEV)[None]
    if not batched:
        k, v, slots = k[0], v[0], slots[0]
    pages = [torch.zeros(3, 16, 2, 64, device=DEV) for _ in range(2)]
    weight = torch.ones(64, device=DEV, requires_grad=True)
    products = [(x * weight).sum() for x in pages]
    append_tokens(k, v, *pages, slots)
    assert all(x._version > 0 for x in pages)
    for product in products:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
    with torch.inference_mode():      # tensors without a version
        cache = [x.clone() for x in pages]
        append_tokens(k, v, *cache, slots + 5)
    append_tokens(k, v, *cache, slots + 9)
    assert torch.equal(cache[0].view(-1, 2, 64)[9:13], k.view(-1, 2, 64))


@pytest.mark.parametrize("batched", [False, True])
@pytest.mark.parametrize("which", range(4))
def test_append_refuses_to_drop_a_gradient(which, batched):
    k, v = (torch.randn(1, 4, 2, 64, device=DEV) for _ in range(2))
    slots = torch.arange(4, device=DEV)[None]
    if not batched:
        k, v, slots = k[0], v[0], slots[0]
    args = [k, v, *(torch.zeros(3, 16, 2, 64, device=DEV) for _ in range(2))]
    args[which].requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        append_tokens(*args, slots)
    assert not args[2].any()
    with torch.no_grad():
        append_tokens(*args, slots)
    assert torch.equal(args[2].view(-1, 2, 64)[:4], k.view(-1, 2, 64))


@pytest.mark.parametrize("drafted,heads", [(2, 8), (20, 4), (40, 16)])
@pytest.mark.parametrize("scale", [-0.3, -1.5, 0.0, -1e-30])
def test_signs_and_zeros_of_the_scale(drafted, heads, scale):
    """8, 40 and 320 rows of a key head, over a cache that several CTAs share."""

    cache = _cache((2500, 90), 16, 2, 64, BF16)
    q, k, v = _fresh(2, drafted, heads, 2, 64, BF16)
    mask = _tree(2, drafted)
    out = tree_attention(q, k, v, *cache, mask, scale=scale)
    _check(out, q, k, v, cache, mask, scale or 1e-300)      # (_check takes a scale of 0 for none; 1e-300 weighs all alike, too)
    assert torch.equal(out, tree_attention(-q, k, v, *cache, mask, scale=-scale))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("drafted,heads,cached", [(9, 4, 40), (200, 4, (130, 1000)), (2500, 2, (60, 700)), (4300, 2, (0,))])
def test_drafts_that_are_not_finite_in_long_chains(dtype, drafted, heads, cached):
    """Values that are not finite reach the channels and rows that see them, and not one bit of anything else, in chains of more
    tokens than are told apart at once, too."""

    cached = (cached,) if isinstance(cached, int) else cached
    cache = _cache(cached, 16, 2, 64, dtype)
    q, k, v = _fresh(len(cached), drafted, heads, 2, 64, dtype)
    clean = tree_attention(q, k, v, *cache)
    reached = torch.zeros_like(clean, dtype=torch.bool)
    nan = torch.zeros_like(reached)
    group = heads // 2
    for b, token, head, channel, what in ((0, drafted - 1, 0, 3, math.nan), (0, drafted // 2, 1, 40, math.inf), (len(cached) - 1, 5, 0, 63, -math.inf),
                                          (0, drafted // 2 + 1, 1, 40, -math.inf), (0, drafted // 3, 1, 8, math.nan)):
        v[b, token, head, channel] = what
        at = (b, slice(token, drafted), slice(head * group, (head + 1) * group), channel)
        nan[at] |= reached[at] | math.isnan(what)
        reached[at] = True
    out = tree_attention(q, k, v, *cache)
    assert torch.equal(out[~reached], clean[~reached])
    assert torch.isnan(out[nan]).all() and torch.isinf(out[reached & ~nan]).all()
