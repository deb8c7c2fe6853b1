"""GPU tests of attention with a sliding window and sinks (forward and gradients) against plain attention in 64 bits, within
bounds that follow from what the kernels round (tests/attention_bounds.py)."""

from __future__ import annotations

import math

import pytest
import torch

import attention_bounds as exact
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen
from gdn2_sm120_b200.window import window_attention, window_attention_varlen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(lead, heads, kv_heads, dim, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(*lead, h, dim, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads, kv_heads, heads)]


def _seen(time, window, sinks):
    i, j = torch.arange(time, device=DEV)[:, None], torch.arange(time, device=DEV)
    return (j <= i) & ((i - j < window) | (j < sinks))


def _check_sequence(got, q, k, v, do, window, sinks, label, scale=None):
    """got: (o, dq, dk, dv) of one sequence, [T, H, D] each"""

    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want = exact.attention(*(x.transpose(0, 1) for x in (q, k, v)), _seen(q.shape[0], window, sinks), scale, do.transpose(0, 1))
    for name, x in zip(("o", "dq", "dk", "dv"), got):
        exact.check(f"{label} {name}", x, *want[name])


def _run(q, k, v, do, window, sinks, bounds=None, scale=None):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    if bounds is None:
        out = window_attention(*leaves, window, sinks=sinks, scale=scale)
    else:
        out = window_attention_varlen(*leaves, bounds, window, sinks=sinks, scale=scale)
    return out.detach(), *torch.autograd.grad(out, leaves, do)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("time,window,sinks,heads,kv_heads,dim", [
    (2, 1, 0, 1, 1, 64), (70, 1, 1, 2, 1, 128), (130, 1, 0, 2, 2, 64), (129, 128, 0, 4, 2, 128), (300, 7, 3, 2, 1, 40),
    (256, 128, 128, 2, 1, 64), (257, 128, 1, 4, 4, 96), (513, 256, 130, 3, 1, 128), (640, 127, 0, 2, 1, 128), (640, 129, 0, 2, 1, 64),
    (700, 300, 5, 8, 1, 128), (900, 200, 0, 2, 2, 72), (1000, 64, 300, 4, 2, 64), (1100, 385, 384, 2, 1, 128), (1500, 130, 2000, 2, 1, 64),
    (1500, 1, 4, 2, 1, 128), (1400, 511, 64, 6, 2, 64),
])
def test_batch_forward_and_gradients(dtype, time, window, sinks, heads, kv_heads, dim):
    batch = 1 + time % 2
    q, k, v, do = _inputs((batch, time), heads, kv_heads, dim, dtype, seed=time + window)
    got = _run(q, k, v, do, window, sinks)
    inference = window_attention(q, k, v, window, sinks=sinks)
    assert torch.equal(inference, got[0]) and inference.is_contiguous()
    for b in range(batch):
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], do[b], window, sinks, f"sequence {b}")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,window,sinks,heads,kv_heads,dim", [
    ((0, 5, 0, 0, 130, 1, 0), 4, 1, 4, 2, 128), ((128, 256, 64, 1, 1, 383), 100, 0, 2, 1, 64), ((1000, 3, 500), 256, 16, 3, 3, 96),
    ((40, 800, 129, 128, 127), 128, 140, 2, 1, 128), ((300,) * 3 + (2,) * 5 + (700,), 33, 2, 4, 1, 64),
])
def test_packed_forward_and_gradients(dtype, lengths, window, sinks, heads, kv_heads, dim):
    bounds = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    q, k, v, do = _inputs((1, bounds[-1]), heads, kv_heads, dim, dtype, seed=7)
    got = _run(q, k, v, do, window, sinks, bounds)
    assert torch.equal(window_attention_varlen(q, k, v, torch.tensor(bounds), window, sinks=sinks), got[0])
    for lo, hi in zip(bounds, bounds[1:]):
        if hi > lo:
            part = slice(lo, hi)
            _check_sequence([x[0, part] for x in got], q[0, part], k[0, part], v[0, part], do[0, part], window, sinks, f"rows {lo} to {hi}")


@pytest.mark.parametrize("lengths,window,sinks,heads,kv_heads,dim", [
    ((1300,), 1100, 0, 12, 1, 64), ((2000,), 130, 4, 16, 1, 128), ((2000,), 130, 300, 8, 1, 40), ((600, 30, 1, 1513), 400, 20, 12, 1, 128),
])
def test_key_gradients_summed_by_several_ctas(lengths, window, sinks, heads, kv_heads, dim):
    """Few sequences and key heads, large groups: the sums of a key's gradients are cut into parts, those of the sinks into
    their own."""

    bounds = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    q, k, v, do = _inputs((1, bounds[-1]), heads, kv_heads, dim, BF16, seed=17)
    got = _run(q, k, v, do, window, sinks, bounds)
    for lo, hi in zip(bounds, bounds[1:]):
        part = slice(lo, hi)
        _check_sequence([x[0, part] for x in got], q[0, part], k[0, part], v[0, part], do[0, part], window, sinks, f"rows {lo} to {hi}")
    assert all(torch.equal(a, b) for a, b in zip(got, _run(q, k, v, do, window, sinks, bounds)))
    if len(lengths) == 1:
        assert all(torch.equal(a, b) for a, b in zip(got, _run(q, k, v, do, window, sinks)))


def test_more_sequences_than_a_launch_holds():
    lengths = [(7 * i) % 61 + (400 if i in (3, 300, 590) else 0) for i in range(600)]
    bounds = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    q, k, v, do = _inputs((1, bounds[-1]), 8, 1, 64, BF16, seed=3)
    got = _run(q, k, v, do, 20, 9, bounds)
    for i in (0, 1, 3, 255, 256, 257, 300, 511, 512, 590, 599):
        part = slice(bounds[i], bounds[i + 1])
        if lengths[i]:
            _check_sequence([x[0, part] for x in got], q[0, part], k[0, part], v[0, part], do[0, part], 20, 9, f"sequence {i}")


@pytest.mark.parametrize("window", [300, 1000, 2 ** 31, 2 ** 70])
def test_a_window_over_everything_is_causal_attention(window):
    q, k, v, do = _inputs((2, 300), 4, 2, 64, BF16, seed=1)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = causal_attention(*leaves)
    want = (out.detach(), *torch.autograd.grad(out, leaves, do))
    for sinks in (0, 7, 2 ** 40):
        assert all(torch.equal(a, b) for a, b in zip(want, _run(q, k, v, do, window, sinks)))
    bounds = (0, 20, 300)
    assert torch.equal(window_attention_varlen(q[:1], k[:1], v[:1], bounds, window), causal_attention_varlen(q[:1], k[:1], v[:1], bounds))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("time,window,sinks,heads,kv_heads,dim", [
    (1, 1, 0, 2, 1, 64), (1, 5, 2 ** 40, 2, 2, 128), (2, 2, 1, 4, 2, 40), (5, 2 ** 70, 3, 2, 1, 128), (127, 127, 200, 2, 1, 64), (128, 500, 0, 4, 1, 96),
    (129, 129, 4, 2, 2, 128), (255, 256, 0, 8, 1, 64), (256, 256, 9, 2, 1, 128), (257, 257, 9, 2, 1, 128),
])
def test_a_window_over_short_sequences(dtype, time, window, sinks, heads, kv_heads, dim):
    q, k, v, do = _inputs((3, time), heads, kv_heads, dim, dtype, seed=time)
    got = _run(q, k, v, do, window, sinks)
    assert torch.equal(window_attention(q, k, v, window, sinks=sinks), got[0])
    for b in range(3):
        _check_sequence([x[b] for x in got], q[b], k[b], v[b], do[b], min(window, time), min(sinks, time), f"sequence {b}")
    lengths = [time, 0, time // 2, 1, time]
    bounds = [sum(lengths[:i]) for i in range(6)]
    q, k, v, do = _inputs((1, bounds[-1]), heads, kv_heads, dim, dtype, seed=time + 1)
    got = _run(q, k, v, do, window, sinks, bounds)
    for i, length in enumerate(lengths):
        part = slice(bounds[i], bounds[i + 1])
        if length:
            _check_sequence([x[0, part] for x in got], q[0, part], k[0, part], v[0, part], do[0, part], min(window, time), min(sinks, time), f"packed sequence {i}")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("time,window", [(3, 3), (3, 2), (11, 11), (11, 100), (100, 100), (100, 20), (600, 4)])
def test_gradients_of_few_keys_are_off_by_two_roundings(dtype, time, window):
    # dq and dk sum products of dS, which is rounded once, and are rounded once: the square root of two roundings in the 2-norm,
    # where a rounding of dS, whose values may lie elsewhere between two powers of two, is one of dq to a sixth (1 / sqrt(12) of
    # a step that is 2^-8 .. 2^-7 of the value): sqrt(1 + (7/6)^2) = 1.54, and 1.65 with a share for P, the statistics and the
    # order of 100000 samples.  Delta from the rounded output alone adds a rounding of that for every key: 1.8 to 2.3 with few of them.
    heads, dim = 8, 64
    batch = max(1, 2400 // time)
    q, k, v, do = _inputs((batch, time), heads, heads, dim, dtype, seed=5)
    got = _run(q, k, v, do, window, 0)
    leaves = [x.double().transpose(1, 2).requires_grad_(True) for x in (q, k, v)]
    scores = (leaves[0] @ leaves[1].transpose(-1, -2) * dim ** -0.5).masked_fill(~_seen(time, window, 0), -math.inf)
    want = torch.autograd.grad(scores.softmax(-1) @ leaves[2], leaves, do.double().transpose(1, 2))
    for name, x, y in zip(("dq", "dk"), got[1:3], want):
        y = y.transpose(1, 2)
        rounding = (y.to(dtype).double() - y).norm()
        assert (x.double() - y).norm() < 1.65 * rounding, name


@pytest.mark.parametrize("sinks", [599, 600, 2 ** 33])
def test_sinks_over_everything_see_all(sinks):
    q, k, v, do = _inputs((1, 600), 2, 1, 64, FP16, seed=2)
    got = _run(q, k, v, do, 5, sinks)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], do[0], 600, 0, "all")


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
def test_scales(scale):
    q, k, v, do = _inputs((1, 400), 2, 1, 64, BF16, seed=5)
    got = _run(q, k, v, do, 100, 3, scale=scale)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], do[0], 100, 3, f"scale {scale}", scale)


@pytest.mark.parametrize("height", [-900.0, -60.0, 60.0, 900.0])
@pytest.mark.parametrize("window,sinks", [(100, 0), (300, 4)])
def test_maxima_that_move_far(height, window, sinks):
    """Scores that rise or fall by `height` from one end of the sequence to the other, and sinks far above or below the rest:
    what a row does not see must not enter its maximum."""

    time, dim = 800, 64
    q, k, v, do = _inputs((1, time), 2, 1, dim, BF16, seed=9)
    # whole numbers times powers of two: the scores are exact in 32 bits
    ramp = (torch.arange(time, device=DEV) // 50).float() * (height / 16 / 4)
    q[..., 0], k[..., 0] = 4.0, ramp[None, :, None].to(BF16)
    k[:, :sinks, :, 0] = 100.0 if height < 0 else -100.0
    got = _run(q, k, v, do, window, sinks, scale=1.0)
    _check_sequence([x[0] for x in got], q[0], k[0], v[0], do[0], window, sinks, f"height {height}", 1.0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_views_of_one_projection(dtype):
    batch, time, heads, kv_heads, dim = 2, 350, 4, 2, 64
    gen = torch.Generator(device=DEV).manual_seed(1)
    fused = torch.randn(batch, time, (heads + 2 * kv_heads) * dim + 8, generator=gen, device=DEV).to(dtype)
    q, k, v = (fused[..., a * dim:b * dim].unflatten(-1, (-1, dim)) for a, b in
               ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
    do = torch.randn(batch, heads, time, dim, generator=gen, device=DEV).to(dtype).transpose(1, 2)   # another order
    got = _run(q, k, v, do, 150, 3)
    assert all(torch.equal(a, b) for a, b in zip(got, _run(*(x.contiguous() for x in (q, k, v, do)), 150, 3)))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("time,window,sinks,row", [
    (700, 200, 0, 300), (700, 200, 4, 300), (700, 200, 4, 2), (700, 200, 4, 4), (700, 200, 4, 127), (700, 1, 0, 130), (700, 128, 0, 256),
    (700, 129, 0, 255), (700, 60, 0, 140), (900, 300, 140, 139), (900, 300, 140, 140), (900, 300, 140, 250), (900, 520, 8, 383), (140, 100, 0, 139),
])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(value, time, window, sinks, row):
    """and not one bit of anything else."""

    q, k, v, _ = _inputs((2, time), 4, 2, 96, BF16, seed=row)
    clean = window_attention(q, k, v, window, sinks=sinks)
    v = v.clone()
    v[1, row, 1, 77] = value
    out = window_attention(q, k, v, window, sinks=sinks)
    reached = torch.zeros_like(out, dtype=torch.bool)
    reached[1, :, 2:, 77] = _seen(time, window, sinks)[:, row, None]
    assert torch.equal(out[~reached], clean[~reached])
    assert not torch.isfinite(out[reached]).any() and (not math.isnan(value) or torch.isnan(out[reached]).all())


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP16, 64)])
def test_many_values_that_are_not_finite(dtype, dim):
    """Several items of a CTA are done once more, packed and not."""

    batch, time, window, sinks = 8, 700, 190, 130
    q, k, v, _ = _inputs((batch, time), 32, 8, dim, dtype, seed=4)
    bounds = [i * time for i in range(batch + 1)]
    packed = [x.reshape(1, -1, *x.shape[2:]) for x in (q, k)]
    clean = window_attention(q, k, v, window, sinks=sinks)
    v = v.clone()
    reached = torch.zeros_like(clean, dtype=torch.bool)
    seen = _seen(time, window, sinks)
    for b in range(0, batch, 2):
        for row in (0, 1, 127, 128, 129, 130, 200, 255, 256, 511, 512, 640, 699):
            head, channel = (b + row) % 8, (7 * row) % dim
            v[b, row, head, channel] = (math.nan, math.inf, -math.inf)[row % 3]
            reached[b, :, 4 * head:4 * head + 4, channel] |= seen[:, row, None]
    out = window_attention(q, k, v, window, sinks=sinks)
    also = window_attention_varlen(*packed, v.reshape(1, -1, 8, dim), bounds, window, sinks=sinks).view(out.shape)
    for x in (out, also):
        assert torch.equal(x[~reached], clean[~reached]) and not torch.isfinite(x[reached]).any()


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_packed_sequences_do_not_see_each_other(what):
    bounds = (0, 200, 365, 500)
    q, k, v, do = _inputs((1, 500), 2, 1, 64, BF16, seed=4)
    want = _run(q, k, v, do, 90, 20, bounds)
    for lo, hi in ((0, 200), (365, 500)):
        inputs = [x.clone() for x in (q, k, v, do)]
        for x in inputs:
            x[:, lo:hi] = what
        got = _run(*inputs, 90, 20, bounds)
        assert all(torch.equal(a[:, 200:365], b[:, 200:365]) for a, b in zip(got, want))


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("at", [2, 300])
def test_gradients_far_from_a_value_that_is_not_finite(which, value, at):
    """Two tiles beyond what sees it or is seen with it, gradients are as they were."""

    time, window, sinks, tile = 1300, 100, 4, 128
    q, k, v, do = _inputs((1, time), 2, 1, 64, BF16, seed=3)
    clean = _run(q, k, v, do, window, sinks)
    tensors = dict(q=q, k=k, v=v, do=do)
    tensors[which] = tensors[which].clone()
    tensors[which][0, at, 0, 5] = value
    got = _run(*tensors.values(), window, sinks)
    rows = torch.arange(time, device=DEV)
    near = (rows - at).abs() < window + 2 * tile
    if which in ("k", "v"):
        if at < sinks:
            return      # every row sees a sink
        untouched = {1: ~near, 2: ~near & (rows >= tile), 3: ~near & (rows >= tile)}   # its rows see the sinks too
    else:
        untouched = {1: ~near, 2: ~near & (rows >= tile), 3: ~near & (rows >= tile)}
    for i, rows in untouched.items():
        assert torch.equal(got[i][0, rows], clean[i][0, rows])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gradients_against_differences(dtype):
    """Along a random direction the gradients give what differences of the loss in 64 bits do."""

    time, heads, dim, window, sinks = 350, 2, 64, 120, 5
    q, k, v, do = _inputs((1, time), heads, 1, dim, dtype, seed=8)
    grads = _run(q, k, v, do, window, sinks)[1:]
    args = [x[0].transpose(0, 1) for x in (q, k, v)]
    seen = _seen(time, window, sinks)
    bounds = exact.attention(*args, seen, dim ** -0.5, do[0].transpose(0, 1))

    def loss(q, k, v):
        s = (q @ k.transpose(1, 2) * dim ** -0.5).masked_fill(~seen, -math.inf)
        return (s.softmax(-1) @ v * do[0].double().transpose(0, 1)).sum()

    h = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(args[i].shape, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV, dtype=torch.float64)
        ends = [[a.double() + (sign * h * way if j == i else 0.0) for j, a in enumerate(args)] for sign in (1, -1)]
        slope = (loss(*ends[0]) - loss(*ends[1])) / (2 * h)
        got = (grads[i][0].transpose(0, 1).double() * way).sum()
        # the third derivative of a softmax of scores of some units, times h^2: far below the gradients' own rounding
        allowed = (bounds[name][1] * way.abs()).sum() + 1e-5 * abs(slope)
        assert abs(got - slope) <= allowed, name


def test_the_same_bits_every_time_alone_and_in_a_batch():
    q, k, v, do = _inputs((3, 633), 4, 2, 128, BF16, seed=6)
    first = _run(q, k, v, do, 200, 4)
    assert all(torch.equal(a, b) for a, b in zip(first, _run(q, k, v, do, 200, 4)))
    alone = _run(q[1:2], k[1:2], v[1:2], do[1:2], 200, 4)
    assert torch.equal(first[0][1:2], alone[0]) and torch.equal(first[1][1:2], alone[1])


def test_another_stream_and_a_captured_training_step():
    q, k, v, do = _inputs((1, 400), 4, 2, 64, BF16, seed=13)
    bounds = (0, 50, 51, 400)
    want = _run(q, k, v, do, 60, 3, bounds)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = window_attention_varlen(*leaves, bounds, 60, sinks=3)
        got = (out.detach(), *torch.autograd.grad(out, leaves, do))
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_attention_varlen(*leaves, bounds, 60, sinks=3)
        grads = torch.autograd.grad(out, leaves, do)
    for seed in (14, 15):
        new = _inputs((1, 400), 4, 2, 64, BF16, seed=seed)
        with torch.no_grad():
            for x, y in zip((*leaves, do), new):
                x.copy_(y)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip((out.detach(), *grads), _run(*new, 60, 3, bounds)))


def test_no_tokens():
    q, k, v, _ = _inputs((2, 0), 4, 2, 64, BF16)
    q.requires_grad_(True)
    out = window_attention(q, k, v, 3, sinks=1)
    assert out.shape == q.shape
    assert torch.autograd.grad(out.sum(), q)[0].shape == q.shape
    assert window_attention_varlen(q[:1].detach(), k[:1], v[:1], (0, 0), 3).shape == (1, 0, 4, 64)


def test_refusals():
    q, k, v, _ = _inputs((1, 16), 4, 2, 64, BF16)
    with pytest.raises(TypeError, match="dtype"):
        window_attention(q, k.half(), v, 4)
    with pytest.raises(ValueError, match="place of its own"):
        window_attention(q, k[:, :, :1].expand(-1, -1, 2, -1), v, 4)
    with pytest.raises(ValueError):
        window_attention_varlen(q, k, v, (0, 9, 8, 16), 4)
    with pytest.raises(ValueError, match="scale"):
        window_attention(q, k, v, 4, scale=math.inf)
    for window, sinks in ((0, 0), (-1, 0), (4, -1)):
        with pytest.raises(ValueError, match="at least"):
            window_attention(q, k, v, window, sinks=sinks)
