"""GPU tests of the operators of bounded memory together: the example, steps and evictions by turns, both host paths, waits that
run out, a second call while the first one runs."""

from __future__ import annotations

import pathlib
import sys

import pytest
import torch

import attention_bounds as exact
from gdn2_sm120_b200 import _lib
from gdn2_sm120_b200.eviction import evict_tokens, weighed_attention, weighed_attention_varlen, weighed_token_attention
from gdn2_sm120_b200.paged import append_tokens
from gdn2_sm120_b200.window import window_attention, window_attention_varlen, window_tree_attention
from test_attention_failures_gpu import _no_waiting, _right_or_nan

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "examples"))

import bounded_memory as example

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _normal(*shape, seed=0, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def test_a_training_step():
    loss, grads = example.training_step()
    again, same = example.training_step()
    assert torch.isfinite(loss) and loss == again
    assert all(torch.isfinite(g).all() and g.any() for g in grads) and all(torch.equal(a, b) for a, b in zip(grads, same))


def test_a_window_over_pages_that_are_given_back():
    got, tokens, layer, used = example.serve_window(prompt_tokens=150, steps=200, window=50, sinks=3, pages=14)
    assert used <= 1 + 50 // 16 + 2
    q, k, v = layer.project(tokens, None)
    want = window_attention(q, k, v, 50, sinks=3)
    # two roundings of weights and outputs (2^-8 each, independent), in the norm of all tokens
    assert (got - want).float().norm() <= 2.0 ** -6 * want.float().norm()


def test_a_cache_that_is_thinned_out():
    out, lengths = example.serve_evicting()
    assert torch.isfinite(out).all() and out.shape[1] == 350
    assert lengths[0] == 96 and max(lengths) == 127 and lengths.count(96) > 3


def test_steps_and_evictions_by_turns():
    """Three sequences of different lengths; every step against plain attention in 64 bits over what the cache then holds, its
    weights against sums in 64 bits that evictions thin out in the same way."""

    page, keep, kv_heads, heads, dim, steps = 16, 48, 2, 4, 64, 40
    first = (90, 40, 61)
    pages = 60
    k_pages, v_pages = _normal(pages, page, kv_heads, dim, seed=1), _normal(pages, page, kv_heads, dim, seed=2)
    weights = torch.rand(pages, kv_heads, page, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    order = torch.randperm(pages, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).int()
    table = order[:30].view(3, 10).clone()
    spare = order[30:48].view(2, 3, 3)
    lengths = torch.tensor(first, device=DEV, dtype=torch.int32)

    def read(b, x, by_head):
        t = torch.arange(int(lengths[b]), device=DEV)
        where = table[b, t // page].long(), t % page
        return x[where[0], :, where[1]] if by_head else x[where]

    sums = [read(b, weights, True).double() for b in range(3)]      # [tokens, kv heads]
    for step in range(steps):
        if step % 13 == 12:
            before = [read(b, weights, True) for b in range(3)]
            new = spare[step // 13 % 2]
            got = evict_tokens(k_pages, v_pages, weights, table, lengths, new.contiguous(), keep, sinks=2, recent=8)
            assert got.tolist() == [min(n, keep) for n in lengths.tolist()]
            for b in range(3):
                n = int(lengths[b])
                if n > keep:
                    w = before[b].clone()
                    w[:2], w[n - 8:] = torch.inf, torch.inf
                    kept = w.sort(dim=0, descending=True, stable=True).indices[:keep].sort(dim=0).values
                    sums[b] = sums[b].gather(0, kept)
            table = torch.cat([new, table[:, 3:]], 1).contiguous()
            lengths = got
        q, k, v = _normal(3, 1, heads, dim, seed=100 + step), _normal(3, 1, kv_heads, dim, seed=200 + step), _normal(3, 1, kv_heads, dim, seed=300 + step)
        places = lengths.long()[:, None]
        slots = table.long().gather(1, places // page) * page + places % page
        out = weighed_token_attention(q, k, v, k_pages, v_pages, weights, table, lengths, slots)
        for b in range(3):
            keys, values = (torch.cat([read(b, x, False), y[b]]) for x, y in ((k_pages, k), (v_pages, v)))
            want = exact.attention(*(x.transpose(0, 1) for x in (q[b], keys, values)), torch.ones(1, len(keys), device=DEV, dtype=torch.bool), dim ** -0.5)
            exact.check(f"step {step}", out[b], *want["o"])
            s = (q[b, 0].double().view(kv_heads, 2, dim) @ keys.double().permute(1, 2, 0)) * dim ** -0.5
            got = torch.softmax(s, -1).sum(1).T
            sums[b] = torch.cat([sums[b] + got[:-1], got[-1:]])
        append_tokens(k, v, k_pages, v_pages, slots)
        lengths = lengths + 1
        for b in range(3):
            # every step's weights are good to 2^-13, and a sum of 32-bit numbers rounds once a step
            assert (read(b, weights, True) - sums[b]).abs().le(2.0 ** -12 * sums[b]).all()


def _everything():
    q, k, v, do = _normal(1, 300, 4, 64, seed=1), _normal(1, 300, 2, 64, seed=2), _normal(1, 300, 2, 64, seed=3), _normal(1, 300, 4, 64, seed=4)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = window_attention_varlen(*leaves, (0, 3, 200, 300), 50, sinks=2, scale=0.2)
    results = [out.detach(), *torch.autograd.grad(out, leaves, do), window_attention(q, k, v, 70)]
    results += [*weighed_attention(q, k, v), *weighed_attention_varlen(q, k, v, (0, 3, 200, 300))]
    pages, weights = [_normal(20, 16, 2, 64, seed=5 + i) for i in range(2)], torch.rand(20, 2, 16, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV)
    table, length = torch.arange(20, device=DEV, dtype=torch.int32)[None], torch.tensor([133], device=DEV, dtype=torch.int32)
    mask = torch.ones(7, 7, device=DEV, dtype=torch.bool).tril()
    mask[5, 2] = False
    depths = torch.arange(7, device=DEV, dtype=torch.int32)
    results += [window_tree_attention(q[:, :7], k[:, :7], v[:, :7], *pages, table, length, 60, sinks=3),
                window_tree_attention(q[:, :7], k[:, :7], v[:, :7], *pages, table, length, 60, mask, depths, sinks=3)]
    results.append(weighed_token_attention(q[:, :2], k[:, :2], v[:, :2], *pages, weights, table, length, torch.tensor([[133, 134]], device=DEV), decay=0.5))
    results.append(evict_tokens(*pages, weights, table[:, :10], length, table[:, 12:].contiguous(), 100, sinks=1, recent=5))
    return results + [*pages, weights]


def test_native_and_python_host_paths_give_the_same():
    _lib.LAUNCHES[0] = 0
    native = _everything()
    launches = _lib.LAUNCHES[0]
    _lib.LAUNCHES[0] = 0
    _lib.KERNEL_EVENTS = {}      # calls that are timed one by one go through Python
    try:
        python = _everything()
        names = set(_lib.KERNEL_EVENTS)
    finally:
        _lib.KERNEL_EVENTS = None
    assert {"gdn2_window_attention_forward", "gdn2_window_attention_backward", "gdn2_attention_weights", "gdn2_window_tree_attention",
            "gdn2_weighed_token_attention", "gdn2_evict_tokens"} <= names
    assert launches == _lib.LAUNCHES[0] > 0
    assert all(torch.equal(a, b) for a, b in zip(native, python))


@pytest.mark.parametrize("lengths,window,sinks,heads,kv_heads,dim", [((700, 700), 200, 4, 4, 2, 128), ((1500,), 130, 0, 2, 1, 64), ((300, 1, 77), 40, 50, 6, 3, 96)])
def test_waits_of_a_window_that_run_out(lengths, window, sinks, heads, kv_heads, dim):
    total, bounds = sum(lengths), tuple(sum(lengths[:i]) for i in range(len(lengths) + 1))
    q, k, v, do = _normal(1, total, heads, dim, seed=1), _normal(1, total, kv_heads, dim, seed=2), _normal(1, total, kv_heads, dim, seed=3), _normal(1, total, heads, dim, seed=4)
    _right_or_nan(lambda: [window_attention_varlen(q, k, v, bounds, window, sinks=sinks)])
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = window_attention_varlen(*leaves, bounds, window, sinks=sinks)
    _right_or_nan(lambda: torch.autograd.grad(out, leaves, do, retain_graph=True))
    strange = v.clone()
    strange[0, ::97, 0, 3] = torch.inf      # items that are done once more
    with _no_waiting():
        for _ in range(4):
            window_attention_varlen(q, k, strange, bounds, window, sinks=sinks)
        torch.cuda.synchronize()


def test_waits_of_weights_and_steps_that_run_out():
    q, k, v = _normal(1, 900, 8, 64, seed=1), _normal(1, 900, 2, 64, seed=2), _normal(1, 900, 2, 64, seed=3)
    _right_or_nan(lambda: weighed_attention(q, k, v)[1:])
    pages = [_normal(70, 16, 2, 64, seed=5 + i) for i in range(2)]
    table, length = torch.randperm(70, device=DEV).int()[None], torch.tensor([1000], device=DEV, dtype=torch.int32)
    weights = torch.zeros(70, 2, 16, device=DEV)
    slots = torch.tensor([[int(table[0, 1000 // 16]) * 16 + 1000 % 16]], device=DEV)

    def step():
        return [weighed_token_attention(q[:, :1], k[:, :1], v[:, :1], *pages, weights, table, length, slots, decay=0.0), weights.clone()]

    _right_or_nan(step)
    for drafted in (3, 40):
        _right_or_nan(lambda: [window_tree_attention(q[:, :drafted], k[:, :drafted], v[:, :drafted], *pages, table, length, 700, sinks=20)])


def test_two_calls_at_once():
    """On two streams, with caches of their own: workspaces are a call's own."""

    pages = [[_normal(200, 16, 2, 64, seed=10 * j + i) for i in range(2)] for j in range(2)]
    weights = [torch.zeros(200, 2, 16, device=DEV) for _ in range(2)]
    table, lengths = torch.arange(200, device=DEV, dtype=torch.int32).view(2, 100), torch.tensor([1500, 800], device=DEV, dtype=torch.int32)
    q, k, v = _normal(2, 1, 8, 64, seed=1), _normal(2, 1, 2, 64, seed=2), _normal(2, 1, 2, 64, seed=3)
    slots = torch.tensor([[1599], [3199]], device=DEV)
    want = [weighed_token_attention(q, k, v, *pages[j], weights[j], table, lengths, slots, decay=0.0) for j in range(2)]
    kept = [w.clone() for w in weights]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for w in weights:
        w.zero_()
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[j].append(weighed_token_attention(q, k, v, *pages[j], weights[j], table, lengths, slots, decay=0.0))
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(x, want[j]) for x in got[j]) and torch.equal(weights[j], kept[j])


@pytest.mark.slow
def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements, of which the last pages are used; the same in a small cache."""

    page, kv_heads, dim, used = 64, 4, 128, 40
    pages = 2 ** 31 // (page * kv_heads * dim) + 2 * used
    small = [_normal(2 * used, page, kv_heads, dim, seed=1 + i) for i in range(2)]
    small.append(torch.rand(2 * used, kv_heads, page, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV))
    large = [torch.zeros(pages, *x.shape[1:], device=DEV, dtype=x.dtype) for x in small]
    for x, y in zip(large, small):
        x[-2 * used:] = y
    table = torch.randperm(used, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).int().view(2, 20)
    lengths = torch.tensor([1200, 777], device=DEV, dtype=torch.int32)
    q, k, v = _normal(2, 1, 16, dim, seed=5), _normal(2, 1, kv_heads, dim, seed=6), _normal(2, 1, kv_heads, dim, seed=7)
    results = []
    for cache, first in ((small, 0), (large, pages - 2 * used)):
        at = table + first
        slots = at.long().gather(1, lengths.long()[:, None] // page) * page + lengths.long()[:, None] % page
        new = torch.arange(used, used + 10, device=DEV, dtype=torch.int32).view(2, 5) + first
        out = [weighed_token_attention(q, k, v, *cache, at, lengths, slots), window_tree_attention(q, k, v, *cache[:2], at, lengths, 300, sinks=70)]
        append_tokens(k, v, *cache[:2], slots)
        out.append(evict_tokens(*cache, at, lengths, new, 300, sinks=2, recent=30))
        results.append(out + [x[first:] for x in cache])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert not any(x[:-2 * used].any() for x in large)
