"""GPU tests of rotary positions against the rotation in 64 bits: two products and their sum in 32 bits, one rounding."""

from __future__ import annotations

import math

import pytest
import torch

from gdn2_sm120_b200.rotary import apply_rotary, rotary_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _turned(x, cos, sin, at, layout):
    """The rotation in 64 bits and, elementwise, what 32-bit arithmetic and one rounding may be off."""

    pairs = cos.shape[1]
    i = torch.arange(pairs, device=DEV)
    a, b = (i, i + pairs) if layout == "half" else (2 * i, 2 * i + 1)
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    xa, xb = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    size[..., a], size[..., b] = (xa * c).abs() + (xb * s).abs(), (xb * c).abs() + (xa * s).abs()
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    turned = size > 0
    return y, torch.where(turned, 1.01 * UNIT[x.dtype] * y.abs() + 2.0 ** -22 * size + tiny, 0.0)


def _inputs(batch, time, heads, kv_heads, dim, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(batch, time, h, dim, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("batch,time,heads,kv_heads,dim,rotated", [
    (1, 1, 1, 1, 2, 2), (2, 3, 5, 1, 128, 128), (3, 17, 32, 8, 128, 64), (1, 100, 7, 3, 96, 48), (2, 9, 4, 4, 80, 24),
    (1, 33, 3, 2, 10, 6), (2, 5, 1, 1, 512, 256), (1, 4, 300, 1, 64, 64), (1, 2, 2, 1, 510, 2),
])
def test_forward_and_gradient(dtype, layout, batch, time, heads, kv_heads, dim, rotated):
    table = 200
    cos, sin = rotary_tables(table, rotated)
    gen = torch.Generator(device=DEV).manual_seed(5)
    at = torch.randint(0, table, (batch, time), generator=gen, device=DEV)
    q, k = (x.requires_grad_(True) for x in _inputs(batch, time, heads, kv_heads, dim, dtype))
    out = apply_rotary(q, k, cos, sin, at, layout=layout)
    cotangents = _inputs(batch, time, heads, kv_heads, dim, dtype, seed=3)
    grads = torch.autograd.grad(out, (q, k), cotangents)
    for got, x, s in zip((*out, *grads), (q, k, *cotangents), (sin, sin, -sin, -sin)):
        want, bound = _turned(x.detach(), cos, s, at, layout)
        assert got.shape == x.shape and got.dtype == dtype
        assert ((got.detach().double() - want).abs() <= bound).all()
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(out, apply_rotary(q, k, cos, sin, at.int(), layout=layout)))
        a, b = q.detach().clone(), k.detach().clone()
        turned = apply_rotary(a, b, cos, sin, at, layout=layout, inplace=True)
        assert turned[0] is a and turned[1] is b and torch.equal(a, out[0]) and torch.equal(b, out[1])


def test_gradient_against_differences():
    """The rotation is linear: a difference of it along a direction is exact up to rounding."""

    cos, sin = rotary_tables(50, 32)
    q, k = _inputs(1, 50, 2, 1, 64, torch.float32)
    cotangents = _inputs(1, 50, 2, 1, 64, torch.float32, seed=1)
    ways = _inputs(1, 50, 2, 1, 64, torch.float32, seed=2)
    q.requires_grad_(True)
    k.requires_grad_(True)
    grads = torch.autograd.grad(apply_rotary(q, k, cos, sin), (q, k), cotangents)
    at = torch.arange(50, device=DEV)[None]
    for x, way, grad, ct in zip((q, k), ways, grads, cotangents):
        ends = [_plain64(x.detach().double() + h * way.double(), cos, sin, at) for h in (0.5, -0.5)]
        slope = ((ends[0] - ends[1]) * ct.double()).sum()
        got = (grad.double() * way.double()).sum()
        assert abs(got - slope) <= 2.0 ** -20 * (grad.double() * way.double()).abs().sum()


def _plain64(x, cos, sin, at):
    pairs = cos.shape[1]
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    a, b, rest = x[..., :pairs], x[..., pairs:2 * pairs], x[..., 2 * pairs:]
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1)


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_views_of_one_projection(offset):
    """Slices of a fused projection, aligned to 16 bytes, to 8 and to 2."""

    batch, time, heads, kv_heads, dim = 2, 11, 4, 2, 64
    gen = torch.Generator(device=DEV).manual_seed(0)
    fused = torch.randn(batch, time, (heads + kv_heads) * dim + 8, generator=gen, device=DEV).bfloat16()
    q = fused[..., offset:offset + heads * dim].unflatten(-1, (heads, dim))
    k = fused[..., offset + heads * dim:offset + (heads + kv_heads) * dim].unflatten(-1, (kv_heads, dim))
    cos, sin = rotary_tables(time, 32)
    want = apply_rotary(q.contiguous(), k.contiguous(), cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(apply_rotary(q, k, cos, sin), want))
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k)]     # [B, H, T, D] in memory
    assert all(torch.equal(a, b) for a, b in zip(apply_rotary(*turned, cos, sin), want))
    before = fused.clone()
    apply_rotary(q, k, cos, sin, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(fused[..., :offset], before[..., :offset])
    assert torch.equal(fused[..., offset + (heads + kv_heads) * dim:], before[..., offset + (heads + kv_heads) * dim:])


def test_positions():
    cos, sin = rotary_tables(40, 64)
    q, k = _inputs(2, 7, 2, 1, 128, torch.bfloat16)
    plain = apply_rotary(q, k, cos, sin)
    steps = torch.arange(7, device=DEV)
    for positions in (steps, steps.int(), steps.expand(2, 7), torch.stack([steps, steps], 1)[:, 0]):
        assert all(torch.equal(a, b) for a, b in zip(apply_rotary(q, k, cos, sin, positions), plain))
    wrong = steps.repeat(2, 1)
    wrong[0, 3], wrong[1, 5] = 40, -1
    out = apply_rotary(q, k, cos, sin, wrong)
    for got, want in zip(out, plain):
        bad = torch.zeros(2, 7, device=DEV, dtype=torch.bool)
        bad[0, 3] = bad[1, 5] = True
        assert torch.isnan(got[bad][..., :64]).all() and torch.equal(got[bad][..., 64:], want[bad][..., 64:])
        assert torch.equal(got[~bad], want[~bad])


def test_a_broadcast_cotangent_another_stream_and_no_tokens():
    cos, sin = rotary_tables(16, 64)
    q, k = (x.requires_grad_(True) for x in _inputs(1, 16, 2, 1, 64, torch.float32))
    a, b = apply_rotary(q, k, cos, sin)
    want = torch.autograd.grad((a, b), (q, k), (torch.ones_like(a), torch.zeros_like(b)), retain_graph=True)
    got = torch.autograd.grad(a.sum(), (q, k), allow_unused=True)
    assert torch.equal(got[0], want[0]) and (got[1] is None or not got[1].any())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.no_grad():
        other = apply_rotary(q, k, cos, sin)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other[0], a) and torch.equal(other[1], b)
    assert apply_rotary(q[:, :0], k[:, :0], cos, sin)[0].shape == (1, 0, 2, 64)


def test_tables():
    cos, sin = rotary_tables(5000, 64, base=500.0)
    speed = 500.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    angle = torch.arange(5000, dtype=torch.float64)[:, None] * speed
    # angles of up to 5000 in 64 bits: their cosines are right to 1e-12, then rounded once
    assert (cos.cpu().double() - angle.cos()).abs().max() < 2.0 ** -24 and (sin.cpu().double() - angle.sin()).abs().max() < 2.0 ** -24
    half = rotary_tables(5000, 64, base=500.0, scaling="linear", factor=2.0)
    assert torch.equal(half[0][::2], cos[:2500]) and torch.equal(half[1][::2], sin[:2500])
    ntk = rotary_tables(100, 64, scaling="ntk", factor=4.0)
    plain = rotary_tables(100, 64)
    assert torch.equal(ntk[1][:, 0], plain[1][:, 0])                       # the fastest pair as before
    slowest = 10000.0 ** (-31 / 32) / 4.0                                  # the slowest four times as slow
    assert (ntk[1][:, -1].double().cpu() - (torch.arange(100).double() * slowest).sin()).abs().max() < 1e-7
    amplitude = 1.0 + 0.1 * math.log(8.0)
    yarn = rotary_tables(100, 64, scaling="yarn", factor=8.0, trained=4096)
    assert torch.allclose(yarn[1][:, 0], plain[1][:, 0] * amplitude, atol=1e-6)
    assert torch.allclose(yarn[0][::8, -1], rotary_tables(100, 64, scaling="linear", factor=8.0)[0][::8, -1] * amplitude, atol=1e-6)


def _good():
    q, k = _inputs(2, 8, 4, 2, 64, torch.bfloat16)
    cos, sin = rotary_tables(8, 64)
    return dict(q=q, k=k, cos=cos, sin=sin, positions=torch.arange(8, device=DEV))


@pytest.mark.parametrize("name,change,error", [
    ("q", lambda x: x[0], ValueError), ("q", lambda x: x.half(), TypeError), ("k", lambda x: x[:, :4], ValueError), ("q", lambda x: None, TypeError),
    ("k", lambda x: x[..., :32], ValueError), ("q", lambda x: x.transpose(2, 3).contiguous().transpose(2, 3), ValueError),
    ("k", lambda x: x.cpu(), ValueError), ("cos", lambda x: x.double(), TypeError), ("sin", lambda x: x[:4], ValueError),
    ("cos", lambda x: x.cpu(), ValueError), ("positions", lambda x: x.float(), TypeError), ("positions", lambda x: x[:4], ValueError),
    ("positions", lambda x: x.cpu(), ValueError), ("positions", lambda x: [0, 1], TypeError), ("q", lambda x: x[:, :, :0], ValueError),
])
def test_refusals(name, change, error):
    args = _good()
    args[name] = change(args[name])
    with pytest.raises(error):
        apply_rotary(**args)


def test_other_refusals():
    args = _good()
    with pytest.raises(ValueError, match="layout"):
        apply_rotary(**args, layout="other")
    with pytest.raises(ValueError, match="more channels"):
        apply_rotary(args["q"], args["k"], *rotary_tables(8, 66))
    with pytest.raises(ValueError, match="fewer positions"):
        apply_rotary(args["q"], args["k"], *rotary_tables(7, 64))
    with pytest.raises(ValueError, match="place"):
        apply_rotary(args["q"], args["k"][:, :, :1].expand(-1, -1, 2, -1), args["cos"], args["sin"], inplace=True)
    args["q"].requires_grad_(True)
    with pytest.raises(ValueError, match="gradient"):
        apply_rotary(**args, inplace=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("batch,time,heads,kv_heads,dim,rotated", [
    # 8 channels at a time (fp32: 4), 4 and 1; the last thread's heads, a block's last token and a call's last block are not full
    (3, 201, 20, 5, 128, 64), (1, 1501, 11, 2, 40, 24), (1, 6007, 3, 2, 10, 6),
    # every thread takes ten heads
    (1, 9001, 37, 6, 128, 128),
    # at the border of one unit a thread: 37 tokens of 12 heads of 256 units are 113664, 38 are more
    (1, 37, 11, 1, 512, 2), (1, 38, 11, 1, 512, 2),
])
def test_many_tokens(dtype, layout, batch, time, heads, kv_heads, dim, rotated):
    table = 300
    cos, sin = rotary_tables(table, rotated)
    gen = torch.Generator(device=DEV).manual_seed(6)
    at = torch.randint(0, table, (batch, time), generator=gen, device=DEV)
    at[-1, -1] = table   # a position outside
    q, k = _inputs(batch, time, heads, kv_heads, dim, dtype)
    for got, x in zip(apply_rotary(q, k, cos, sin, at, layout=layout), (q, k)):
        assert got[-1, -1, :, :rotated].isnan().all() and torch.equal(got[-1, -1, :, rotated:], x[-1, -1, :, rotated:])
        want, bound = _turned(x, cos, sin, at.clamp(max=table - 1), layout)
        inside = torch.ones(batch, time, dtype=torch.bool, device=DEV)
        inside[-1, -1] = False
        assert ((got.double() - want).abs() <= bound)[inside].all()


def test_in_place_refuses_tensors_that_share_elements():
    cos, sin = rotary_tables(8, 64)
    fused = torch.randn(2, 8, 6 * 64, device=DEV).bfloat16()
    q, k = fused[..., :4 * 64].unflatten(-1, (4, 64)), fused[..., 4 * 64:].unflatten(-1, (2, 64))
    before = fused.clone()
    for a, b in (
        (q, q), (k, k), (q, q[:, :, 3:]),                                             # the same, or one with a part of it
        (q, fused[..., 3 * 64 + 62:5 * 64 + 62].unflatten(-1, (2, 64))),              # two channels in common
        (fused.as_strided((2, 8, 5, 64), (6 * 64 * 8, 6 * 64, 62, 1)), k[:1].expand(2, -1, -1, -1).clone()),
        (q.contiguous(), k[:, :1].expand(-1, 8, -1, -1)),
    ):
        with pytest.raises(ValueError, match="places of their own"):
            apply_rotary(a, b, cos, sin, inplace=True)
    with pytest.raises(ValueError, match="do not lie in"):
        whole = torch.randn(2, 8, 4, 64, device=DEV)
        apply_rotary(whole, whole[:, :, :2].clone(), whole.view(-1)[:256].view(8, 32), sin, inplace=True)
    assert torch.equal(fused, before)
    want = apply_rotary(q, k, cos, sin)
    assert apply_rotary(q, k, cos, sin, inplace=True)[0] is q
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    # heads of q and k by turns, and halves of a batch
    pairs = torch.randn(2, 8, 3, 2, 64, device=DEV)
    want = apply_rotary(pairs[..., 0, :], pairs[..., 1, :], cos, sin)
    apply_rotary(pairs[..., 0, :], pairs[..., 1, :], cos, sin, inplace=True)
    assert torch.equal(pairs[..., 0, :], want[0]) and torch.equal(pairs[..., 1, :], want[1])


def test_in_place_is_seen_by_autograd():
    """A tensor that a backward has saved and that is turned afterwards gives an error, and no wrong gradient."""

    cos, sin = rotary_tables(8, 64)
    q, k = _inputs(2, 8, 4, 2, 64, torch.float32)
    weight = torch.ones(64, device=DEV, requires_grad=True)
    product = (k * weight).sum()
    versions = q._version, k._version
    apply_rotary(q, k, cos, sin, inplace=True)
    assert q._version > versions[0] and k._version > versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with torch.inference_mode():      # tensors without a version
        a, b = q.clone(), k.clone()
        want = apply_rotary(a, b, cos, sin)
        apply_rotary(a, b, cos, sin, inplace=True)
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    apply_rotary(a, b, cos, sin, inplace=True)


def test_the_ramp_of_yarn_is_linear_in_a_pairs_turns():
    rotated, base, trained, factor, fast, slow = 128, 10000.0, 4096, 8.0, 32.0, 1.0
    cos, sin = rotary_tables(2, rotated, base=base, scaling="yarn", factor=factor, trained=trained, fast=fast, slow=slow)
    got = torch.atan2(sin[1].double(), cos[1].double()).cpu()            # an angle of at most 1: that of position 1
    between = 0
    for i in range(rotated // 2):
        speed = base ** (-2.0 * i / rotated)
        turns = trained * speed / (2.0 * math.pi)
        share = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
        between += 0.0 < share < 1.0
        want = share * speed + (1.0 - share) * speed / factor
        # cosine and sine rounded to 32 bits, relative to the amplitude
        assert abs(got[i] - want) <= 2.0 ** -23 * (1.0 + want), i
    assert between > 20
