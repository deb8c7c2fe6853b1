"""GPU tests of causal attention (forward and gradients) against plain attention in 64 bits, within bounds that follow
from what the kernels round (tests/attention_bounds.py)."""

from __future__ import annotations

import math

import pytest
import torch

import attention_bounds as exact
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(lead, heads, kv_heads, dim, dtype, seed=0, size=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(*lead, h, dim, generator=gen, device=DEV) * size).to(dtype) for h in (heads, kv_heads, kv_heads, heads)]


def _check_sequence(got, q, k, v, do, scale, label):
    """got: (o, dq, dk, dv) of one sequence, [T, H, D] each"""

    want = exact.attention(*(x.transpose(0, 1) for x in (q, k, v)), exact.causal(q.shape[0], DEV), scale, do.transpose(0, 1))
    for name, x in zip(("o", "dq", "dk", "dv"), got):
        exact.check(f"{label} {name}", x, *want[name])


def _run(q, k, v, do, bounds=None, scale=None):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = causal_attention(*leaves, scale=scale) if bounds is None else causal_attention_varlen(*leaves, bounds, scale=scale)
    grads = torch.autograd.grad(out, leaves, do)
    for x, g in zip(leaves, grads):
        assert g.shape == x.shape and g.dtype == x.dtype
    return out.detach(), *grads


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("batch,time,heads,kv_heads,dim", [
    (1, 1, 1, 1, 128), (2, 2, 2, 1, 64), (3, 63, 4, 2, 128), (1, 64, 2, 2, 8), (2, 65, 6, 2, 40), (1, 127, 3, 1, 64),
    (2, 128, 2, 1, 128), (1, 129, 4, 4, 72), (1, 255, 2, 2, 128), (2, 256, 2, 1, 96), (1, 257, 8, 1, 128),
    (2, 511, 2, 2, 64), (1, 777, 3, 3, 120), (1, 1500, 2, 1, 128),
])
def test_batch_forward_and_gradients(dtype, batch, time, heads, kv_heads, dim):
    q, k, v, do = _inputs((batch, time), heads, kv_heads, dim, dtype, seed=time)
    got = _run(q, k, v, do)
    inference = causal_attention(q, k, v)
    assert torch.equal(inference, got[0]) and inference.is_contiguous()
    for b in range(batch):
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], do[b], dim ** -0.5, f"sequence {b}")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [
    ((1,), 1, 1, 64), ((0, 5, 0, 0, 130, 1, 0), 4, 2, 128), ((128, 256, 64, 1, 1, 383), 2, 1, 64),
    ((1000, 3, 500), 3, 3, 96),
])
def test_packed_forward_and_gradients(dtype, lengths, heads, kv_heads, dim):
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    q, k, v, do = _inputs((1, bounds[-1]), heads, kv_heads, dim, dtype, seed=7)
    got = _run(q, k, v, do, bounds)
    assert torch.equal(causal_attention_varlen(q, k, v, torch.tensor(bounds)), got[0])
    for lo, hi in zip(bounds, bounds[1:]):
        if hi > lo:
            part = slice(lo, hi)
            _check_sequence([x[0, part] for x in got], q[0, part], k[0, part], v[0, part], do[0, part], dim ** -0.5,
                            f"rows {lo} to {hi}")


@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [((700,), 8, 1, 64), ((1300,), 6, 2, 40), ((600, 30, 1, 513), 12, 1, 128)])
def test_key_gradients_summed_by_several_ctas(lengths, heads, kv_heads, dim):
    """Few sequences and key heads, large groups: the sums of a key's gradients are cut into parts."""

    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    q, k, v, do = _inputs((1, bounds[-1]), heads, kv_heads, dim, BF16, seed=17)
    got = _run(q, k, v, do, bounds)
    for lo, hi in zip(bounds, bounds[1:]):
        part = slice(lo, hi)
        _check_sequence([x[0, part] for x in got], q[0, part], k[0, part], v[0, part], do[0, part], dim ** -0.5, f"rows {lo} to {hi}")
    assert all(torch.equal(a, b) for a, b in zip(got, _run(q, k, v, do, bounds)))
    if len(lengths) == 1:
        assert all(torch.equal(a, b) for a, b in zip(got, _run(q, k, v, do)))


def test_more_sequences_than_a_launch_holds():
    lengths = [(7 * i) % 61 for i in range(600)]
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    q, k, v, do = _inputs((1, bounds[-1]), 2, 1, 64, BF16, seed=3)
    got = _run(q, k, v, do, bounds)
    for i in (0, 1, 255, 256, 257, 511, 512, 599):
        part = slice(bounds[i], bounds[i + 1])
        if lengths[i]:
            _check_sequence([x[0, part] for x in got], q[0, part], k[0, part], v[0, part], do[0, part], 64 ** -0.5, f"sequence {i}")


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
def test_scales(scale):
    q, k, v, do = _inputs((1, 200), 2, 1, 64, BF16, seed=5)
    got = _run(q, k, v, do, scale=scale)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], do[0], scale, f"scale {scale}")


@pytest.mark.parametrize("rising", [True, False])
def test_maxima_that_move_far(rising):
    """Scores that grow (or fall) by some hundred along the keys: the running maximum moves at every tile, or never."""

    time, dim = 700, 64
    q, k, v, do = _inputs((1, time), 2, 1, dim, BF16, seed=9)
    # whole numbers times powers of two: the scores are exact in 32 bits
    ramp = (torch.arange(time, device=DEV) // 64 * (8 if rising else -8)).float()
    q[..., 0], k[..., 0] = 4.0, ramp[None, :, None].to(BF16)
    got = _run(q, k, v, do, scale=1.0)
    want = exact.attention(*(x[0].transpose(0, 1) for x in (q, k, v)), exact.causal(time, DEV), 1.0, do[0].transpose(0, 1))
    # scores of up to 400 in 32 bits are off by 400 * 2^-23 of a power of e, within what the bounds allow for 32 bits
    for name, x in zip(("o", "dq", "dk", "dv"), got):
        exact.check(name, x[0], *want[name])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("height", [20.0, 60.0, 400.0])
def test_single_scores_far_above_all_others(dtype, height):
    """Weights against the reference of earlier tiles would leave the 16-bit types' range, or the 32-bit one's."""

    time, dim = 520, 64
    q, k, v, do = _inputs((1, time), 2, 1, dim, dtype, seed=11)
    q[..., 0], k[..., 0] = 4.0, 0.0
    for at, share in ((3, 0.25), (140, 0.5), (300, 0.75), (301, 0.75), (511, 1.0)):
        k[0, at, 0, 0] = height * share / 4.0
    got = _run(q, k, v, do, scale=1.0)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], do[0], 1.0, f"height {height}")


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_views_of_one_projection_and_gradients_of_views(dtype):
    batch, time, heads, kv_heads, dim = 2, 150, 4, 2, 64
    gen = torch.Generator(device=DEV).manual_seed(1)
    fused = torch.randn(batch, time, (heads + 2 * kv_heads) * dim + 8, generator=gen, device=DEV).to(dtype)
    q, k, v = (fused[..., a * dim:b * dim].unflatten(-1, (-1, dim)) for a, b in
               ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
    do = torch.randn(batch, heads, time, dim, generator=gen, device=DEV).to(dtype).transpose(1, 2)   # another order
    got = _run(q, k, v, do)
    plain = _run(*(x.contiguous() for x in (q, k, v, do)))
    assert all(torch.equal(a, b) for a, b in zip(got, plain))
    # [B, H, T, D] tensors seen as [B, T, H, D]
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert all(torch.equal(a, b) for a, b in zip(_run(*turned, do), plain))


def test_gradient_of_a_broadcast_cotangent_and_of_some_inputs():
    q, k, v, _ = _inputs((1, 90), 2, 1, 64, BF16, seed=2)
    ones = torch.ones_like(q)
    want = _run(q, k, v, ones)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    causal_attention(*leaves).sum().backward()          # the cotangent is an expanded scalar
    assert all(torch.equal(x.grad, g) for x, g in zip(leaves, want[1:]))
    only = v.clone().requires_grad_(True)
    causal_attention(q, k, only).sum().backward()
    assert torch.equal(only.grad, want[3]) and q.grad is None
    # a key shared by expansion: its gradient is the sum over the places it was broadcast to
    shared = k[:, :, :1].clone().requires_grad_(True)
    out = causal_attention(q, shared.expand(-1, -1, 2, -1).contiguous(), v.expand(-1, -1, 2, -1).contiguous())
    assert torch.equal(out, causal_attention(q, k, v))
    out.sum().backward()
    assert shared.grad.shape == shared.shape


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_packed_sequences_do_not_see_each_other(what):
    bounds = (0, 100, 165, 300)
    q, k, v, do = _inputs((1, 300), 2, 1, 64, BF16, seed=4)
    want = _run(q, k, v, do, bounds)
    for lo, hi in ((0, 100), (165, 300)):
        inputs = [x.clone() for x in (q, k, v, do)]
        for x in inputs:
            x[:, lo:hi] = what
        got = _run(*inputs, bounds)
        for a, b in zip(got, want):
            assert torch.equal(a[:, 100:165], b[:, 100:165])


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("time,at", [(300, 0), (300, 129), (300, 255), (300, 299), (70, 33), (600, 260)])
def test_later_tokens_may_hold_anything(what, time, at):
    """A token that is not finite reaches itself and the later ones, and no earlier one."""

    q, k, v, _ = _inputs((1, time), 2, 1, 72, FP16, seed=at)
    want = exact.attention(*(x[0].transpose(0, 1) for x in (q, k, v)), exact.causal(time, DEV), 72 ** -0.5)["o"]
    for which in range(3):
        inputs = [x.clone() for x in (q, k, v)]
        inputs[which][0, at, :, 5] = what
        out = causal_attention(*inputs)
        exact.check("earlier", out[0, :at], *(x[:, :at] for x in want))
        if which == 0:      # a query is its own
            exact.check("later", out[0, at + 1:], *(x[:, at + 1:] for x in want))
            assert torch.isnan(out[:, at]).all()
        elif which == 1 and math.isnan(what):
            assert torch.isnan(out[:, at:]).all()
        elif which == 2:
            assert not torch.isfinite(out[:, at:, :, 5]).any()
            others = [c for c in range(72) if c != 5]
            exact.check("other channels", out[0][..., others], *(x[..., others] for x in want))
            if math.isnan(what):
                assert torch.isnan(out[:, at:, :, 5]).all()


def test_the_same_bits_every_time_alone_and_in_a_batch():
    q, k, v, do = _inputs((3, 333), 4, 2, 128, BF16, seed=6)
    first = _run(q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(first, _run(q, k, v, do)))
    alone = _run(q[1:2], k[1:2], v[1:2], do[1:2])
    assert all(torch.equal(a[1:2], b) for a, b in zip(first, alone))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gradients_against_differences(dtype):
    """Along a random direction the gradients give what differences of the loss in 64 bits do."""

    time, heads, kv_heads, dim = 150, 2, 1, 64
    q, k, v, do = _inputs((1, time), heads, kv_heads, dim, dtype, seed=8)
    grads = _run(q, k, v, do)[1:]
    args = [x[0].transpose(0, 1) for x in (q, k, v)]
    bounds = exact.attention(*args, exact.causal(time, DEV), dim ** -0.5, do[0].transpose(0, 1))

    def loss(q, k, v):
        s = (q @ k.repeat_interleave(heads, 0).transpose(1, 2) * dim ** -0.5).masked_fill(~exact.causal(time, DEV), -math.inf)
        return (s.softmax(-1) @ v.repeat_interleave(heads, 0) * do[0].double().transpose(0, 1)).sum()

    h = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(args[i].shape, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV, dtype=torch.float64)
        ends = [[a.double() + (sign * h * way if j == i else 0.0) for j, a in enumerate(args)] for sign in (1, -1)]
        slope = (loss(*ends[0]) - loss(*ends[1])) / (2 * h)
        got = (grads[i][0].transpose(0, 1).double() * way).sum()
        # the third derivative of a softmax of scores of some units, times h^2: far below the gradients' own rounding
        allowed = (bounds[name][1] * way.abs()).sum() + 1e-5 * abs(slope)
        assert abs(got - slope) <= allowed, name


def test_another_stream_and_a_captured_graph():
    q, k, v, do = _inputs((2, 300), 4, 2, 128, BF16, seed=12)
    want = _run(q, k, v, do)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _run(q, k, v, do)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    causal_attention(q, k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = causal_attention(q, k, v)
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(out, causal_attention(q, k, v))


def test_a_captured_training_step():
    q, k, v, do = _inputs((1, 400), 4, 2, 64, BF16, seed=13)
    bounds = (0, 150, 151, 400)
    _run(q, k, v, do, bounds)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):      # autograd's own first step
        torch.autograd.grad(causal_attention_varlen(*leaves, bounds), leaves, do)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = causal_attention_varlen(*leaves, bounds)
        grads = torch.autograd.grad(out, leaves, do)
    for seed in (14, 15):
        new = _inputs((1, 400), 4, 2, 64, BF16, seed=seed)
        with torch.no_grad():
            for x, y in zip((*leaves, do), new):
                x.copy_(y)
        graph.replay()
        want = _run(*new[:3], new[3], bounds)
        assert all(torch.equal(a, b) for a, b in zip((out.detach(), *grads), want))


def test_no_tokens():
    q, k, v, _ = _inputs((2, 0), 4, 2, 64, BF16)
    q.requires_grad_(True)
    out = causal_attention(q, k, v)
    assert out.shape == q.shape
    assert torch.autograd.grad(out.sum(), q)[0].shape == q.shape
    assert causal_attention_varlen(q[:1].detach(), k[:1], v[:1], (0, 0)).shape == (1, 0, 4, 64)


@pytest.mark.slow
def test_offsets_beyond_32_bits():
    """Queries of more than 2^32 bytes and 2^31 elements; the last sequence is compared."""

    batch, time, heads = 520, 1030, 32
    gen = torch.Generator(device=DEV).manual_seed(0)
    q = torch.empty(batch, time, heads, 128, device=DEV, dtype=BF16).normal_(generator=gen)
    k, v = (torch.empty(batch, time, 1, 128, device=DEV, dtype=BF16).normal_(generator=gen) for _ in range(2))
    out = causal_attention(q, k, v)
    want = causal_attention(q[-1:].clone(), k[-1:].clone(), v[-1:].clone())
    assert torch.equal(out[-1:], want)
    head = exact.attention(q[-1, :, -1:].transpose(0, 1), k[-1].transpose(0, 1), v[-1].transpose(0, 1), exact.causal(time, DEV), 128 ** -0.5)
    exact.check("last head", out[-1, :, -1:], *head["o"])


def _good():
    return _inputs((1, 16), 4, 2, 64, BF16)[:3]


@pytest.mark.parametrize("change,error,match", [
    (lambda q, k, v: (q.float(), k, v), TypeError, "float16 or torch.bfloat16"),
    (lambda q, k, v: (q, k.half(), v), TypeError, "dtype"),
    (lambda q, k, v: (q, k, None), TypeError, "Tensor"),
    (lambda q, k, v: (q[0], k, v), ValueError, "rank-4"),
    (lambda q, k, v: (q, k[:, :8], v[:, :8]), ValueError, "q's"),
    (lambda q, k, v: (q, k, v[:, :, :1]), ValueError, "same shape"),
    (lambda q, k, v: (q[:, :, :3].contiguous(), k, v), ValueError, "multiple"),
    (lambda q, k, v: (q[:, :, :0], k, v), ValueError, "positive"),
    (lambda q, k, v: (q, k.cpu(), v), ValueError, "same device"),
    (lambda q, k, v: tuple(x[..., :60] for x in (q, k, v)), NotImplementedError, "multiples of 8"),
    (lambda q, k, v: tuple(torch.cat([x] * 3, -1) for x in (q, k, v)), NotImplementedError, "up to 128"),
    (lambda q, k, v: tuple(x.transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)), ValueError, "channels"),
    (lambda q, k, v: (q, k[:, :, :1].expand(-1, -1, 2, -1), v), ValueError, "place of its own"),
    (lambda q, k, v: (torch.zeros(q.numel() + 4, device=DEV, dtype=BF16)[4:].view(q.shape), k, v), ValueError, "aligned"),
])
def test_refusals(change, error, match):
    with pytest.raises(error, match=match):
        causal_attention(*change(*_good()))


def test_refusals_of_bounds_and_scales():
    q, k, v = _good()
    for bounds, error in (((0, 8), ValueError), ((1, 16), ValueError), ((0, 9, 8, 16), ValueError), ((0,), ValueError),
                          (torch.zeros(2), TypeError)):
        with pytest.raises(error):
            causal_attention_varlen(q, k, v, bounds)
    with pytest.raises(ValueError, match="shape"):
        causal_attention_varlen(torch.cat([q, q]), torch.cat([k, k]), torch.cat([v, v]), (0, 16))
    for scale in (math.inf, math.nan, 1e60):
        with pytest.raises(ValueError, match="scale"):
            causal_attention(q, k, v, scale=scale)
