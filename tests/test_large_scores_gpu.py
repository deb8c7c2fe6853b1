"""GPU tests of attention with scores that are whole multiples of a power of two and as large as 2^31: exact in 32 bits, so that
the result is that of the formula in 64 bits, within the bounds of any other scores (tests/attention_bounds.py)."""

from __future__ import annotations

import pytest
import torch

import attention_bounds as exact
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen
from gdn2_sm120_b200.paged import tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16
# exponents of the scores on both sides of 1024 powers of two, where the reference changes its form, up to 2^31; the scale
# that multiplies them: scores of 2^28 that lie 1/8 apart, too
HEIGHTS = [(9, 1.0), (10, 1.0), (12, 1.0), (20, 1.0), (28, 1.0), (28, 2.0 ** -8), (31, 1.0), (31, 2.0 ** -9)]


def _scores(q, k, exponent, signs, steps):
    """Sets q [.., H, D] and k [.., Hkv, D] so that q . k = signs 2^exponent + steps 2^(exponent - 23), both per key: two equal
    products and a small one, all of powers of two or times a few bits."""

    q.zero_()
    k.zero_()
    half = (exponent - 1) // 2
    q[..., 0] = q[..., 1] = 2.0 ** half
    k[..., 0] = k[..., 1] = (signs * 2.0 ** (exponent - 1 - half))[..., None].to(k.dtype)
    low = (exponent - 23) // 2
    q[..., 2] = 2.0 ** low
    k[..., 2] = (steps * 2.0 ** (exponent - 23 - low))[..., None].to(k.dtype)


def _keys(count, way, seed=0):
    """Signs and steps of `count` keys: all low, all high, or low ones first; many ties."""

    gen = torch.Generator(device=DEV).manual_seed(seed)
    steps = torch.randint(0, 4, (count,), generator=gen, device=DEV).float()
    signs = torch.ones(count, device=DEV)
    if way == "low":
        signs = -signs
    elif way == "mixed":
        signs[:2 * count // 3] = -1.0
        signs[::97] = 1.0 if count > 97 else -1.0
    return signs, steps


def _normal(shape, dtype, seed, size=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * size).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("exponent,scale", HEIGHTS)
@pytest.mark.parametrize("way", ["high", "low", "mixed"])
@pytest.mark.parametrize("drafted,heads,cached", [(2, 8, 700), (2, 8, 9000), (20, 4, 700), (20, 4, 9000), (40, 16, 700), (40, 16, 5000)])
def test_trees(dtype, exponent, scale, way, drafted, heads, cached):
    """8, 40 and 320 rows of a key head; few tiles, and so many that several CTAs share a sequence."""

    kv_heads, dim, page = 2, 64, 16
    signs, steps = _keys(cached + drafted, way)
    q, v = _normal((1, drafted, heads, dim), dtype, 1), _normal((1, cached + drafted, kv_heads, dim), dtype, 2)
    k = torch.empty_like(v)
    _scores(q, k, exponent, signs, steps)
    pages = -(-cached // page)
    table = torch.randperm(pages, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).int()[None]
    k_pages, v_pages = (torch.zeros(pages, page, kv_heads, dim, device=DEV, dtype=dtype) for _ in range(2))
    t = torch.arange(cached, device=DEV)
    for to, x in ((k_pages, k), (v_pages, v)):
        to[table[0, t // page].long(), t % page] = x[0, :cached]
    out = tree_attention(q, k[:, cached:].contiguous(), v[:, cached:].contiguous(), k_pages, v_pages, table,
                         torch.tensor([cached], device=DEV, dtype=torch.int32), scale=scale)
    seen = torch.cat([torch.ones(drafted, cached, device=DEV, dtype=torch.bool), exact.causal(drafted, DEV)], 1)
    want = exact.attention(*(x[0].transpose(0, 1) for x in (q, k, v)), seen, scale)
    exact.check("tree", out[0], *want["o"])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("exponent,scale", HEIGHTS)
@pytest.mark.parametrize("way", ["high", "low", "mixed"])
@pytest.mark.parametrize("lengths,dim", [((700,), 64), ((1, 130, 520), 128)])
def test_causal(dtype, exponent, scale, way, lengths, dim):
    heads, kv_heads, total = 4, 2, sum(lengths)
    bounds = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    q, v = _normal((1, total, heads, dim), dtype, 4), _normal((1, total, kv_heads, dim), dtype, 5)
    k = torch.empty_like(v)
    _scores(q, k, exponent, *_keys(total, way))
    out = causal_attention(q, k, v, scale=scale) if len(lengths) == 1 else causal_attention_varlen(q, k, v, bounds, scale=scale)
    for lo, hi in zip(bounds, bounds[1:]):
        want = exact.attention(*(x[0, lo:hi].transpose(0, 1) for x in (q, k, v)), exact.causal(hi - lo, DEV), scale)
        exact.check(f"rows {lo} to {hi}", out[0, lo:hi], *want["o"])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("exponent,scale", HEIGHTS)
@pytest.mark.parametrize("way", ["high", "low", "mixed"])
@pytest.mark.parametrize("lengths,heads,dim", [((700,), 4, 64), ((1, 130, 520), 4, 128), ((1100,), 12, 64)])
def test_causal_gradients(dtype, exponent, scale, way, lengths, heads, dim):
    """dq and dk are sums of keys and queries of up to 2^15: small cotangents keep them in fp16's range.  The last lengths have
    the sums over the keys cut into parts."""

    kv_heads, total = 2, sum(lengths)
    bounds = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    q, v = _normal((1, total, heads, dim), dtype, 4), _normal((1, total, kv_heads, dim), dtype, 5)
    do = _normal(q.shape, dtype, 6, 2.0 ** -14)
    k = torch.empty_like(v)
    _scores(q, k, exponent, *_keys(total, way))
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = causal_attention(q, k, v, scale=scale) if len(lengths) == 1 else causal_attention_varlen(q, k, v, bounds, scale=scale)
    grads = torch.autograd.grad(out, leaves, do)
    for lo, hi in zip(bounds, bounds[1:]):
        want = exact.attention(*(x.detach()[0, lo:hi].transpose(0, 1) for x in leaves), exact.causal(hi - lo, DEV), scale,
                               do[0, lo:hi].transpose(0, 1))
        for name, x in zip(("o", "dq", "dk", "dv"), (out.detach(), *grads)):
            exact.check(f"{name}, rows {lo} to {hi}", x[0, lo:hi], *want[name])


@pytest.mark.parametrize("scale,size", [(0.0, 2.0 ** 127), (2.0 ** -130, 2.0 ** 127), (-2.0 ** -126, 2.0 ** 126), (3e38, 0.0), (-3e38, 0.0),
                                        (2.0 ** 127, 2.0 ** -126)])
@pytest.mark.parametrize("drafted,heads", [(2, 8), (20, 4), (40, 16)])
def test_scales_of_any_size(scale, size, drafted, heads):
    """Scores of up to some units from products and scales at the ends of the 32-bit range, and a scale of 0."""

    kv_heads, dim, cached = 2, 64, 300
    total = cached + drafted
    q, v = _normal((1, total, heads, dim), BF16, 1), _normal((1, total, kv_heads, dim), BF16, 2)
    k = torch.zeros_like(v)
    q.zero_()
    steps = torch.randint(-4, 5, (total,), generator=torch.Generator(device=DEV).manual_seed(7), device=DEV) / 4.0
    if size:
        exponent = round(torch.log2(torch.tensor(size)).item())
        q[..., 0] = 2.0 ** (exponent // 2)
        k[..., 0] = (steps * 2.0 ** (exponent - exponent // 2))[:, None].to(BF16)
    want = exact.attention(*(x[0].transpose(0, 1) for x in (q, k, v)), exact.causal(total, DEV), scale)["o"]
    exact.check("causal", causal_attention(q, k, v, scale=scale)[0], *want)
    pages = [torch.zeros(19, 16, kv_heads, dim, device=DEV, dtype=BF16) for _ in range(2)]
    for to, x in zip(pages, (k, v)):
        to.view(-1, kv_heads, dim)[:cached] = x[0, :cached]
    out = tree_attention(*(x[:, cached:].contiguous() for x in (q, k, v)), *pages, torch.arange(19, device=DEV, dtype=torch.int32)[None],
                         torch.tensor([cached], device=DEV, dtype=torch.int32), scale=scale)
    exact.check("tree", out[0], *(x[:, cached:] for x in want))
