"""Full-attention layers whose memory of the past is bounded, in training and in serving.

    python examples/bounded_memory.py

Two ways of it:

  window     a token sees the last tokens and a few first ones (``window_attention_varlen`` in training and for prompts,
             ``window_tree_attention`` over the cache): pages that the window has left are free for others, and
             ``serve_window`` gives them back
  eviction   every token is seen, and what weight it gets is kept count of (``weighed_attention`` for prompts,
             ``weighed_token_attention`` for steps); when the cache is full, ``evict_tokens`` keeps the tokens of the largest weights,
             for every head its own (``serve_evicting``)
"""

from __future__ import annotations

import pathlib
import sys

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))
sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))

from attention_layer import AttentionLayer

from gdn2_sm120_b200.eviction import evict_tokens, weighed_attention, weighed_token_attention
from gdn2_sm120_b200.paged import append_tokens
from gdn2_sm120_b200.window import window_attention, window_attention_varlen, window_tree_attention


def training_step(lengths=(70, 1, 300), window=64, sinks=4, width=256, seed=0):
    """The loss and the gradients of tokens and weights, over packed sequences."""

    gen = torch.Generator(device="cuda").manual_seed(seed)
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    layer = AttentionLayer(width, 4, 2, 64, max(lengths), seed=seed)
    x = torch.randn(1, bounds[-1], width, generator=gen, device="cuda").bfloat16()
    leaves = [x.requires_grad_(True), layer.w_in.requires_grad_(True), layer.w_out.requires_grad_(True)]
    positions = torch.cat([torch.arange(n, device="cuda") for n in lengths])
    q, k, v = layer.project(x, positions)
    out = window_attention_varlen(q, k, v, tuple(bounds), window, sinks=sinks).flatten(-2) @ layer.w_out
    loss = out.float().square().mean()
    return loss.detach(), torch.autograd.grad(loss, leaves)


class Cache:
    """The pages of one sequence, and a pool that they come from and go back to."""

    def __init__(self, layer, pages, page):
        shape = (pages, page, layer.kv_heads, layer.dim)
        self.page = page
        self.keys, self.values = (torch.zeros(shape, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        self.weights = torch.zeros(pages, layer.kv_heads, page, device="cuda")
        self.free = list(range(pages))
        self.table = torch.full((1, 64), -1, device="cuda", dtype=torch.int32)
        self.pages, self.length = [], 0

    def slots(self, count):
        """Places for the next `count` tokens."""

        while len(self.pages) * self.page < self.length + count:
            self.pages.append(self.free.pop())
            self.table[0, len(self.pages) - 1] = self.pages[-1]
        at = torch.arange(self.length, self.length + count, device="cuda")
        return self.table[:, at // self.page].long() * self.page + at % self.page

    def lengths(self):
        return torch.tensor([self.length], device="cuda", dtype=torch.int32)

    def give_back(self, first, last):
        """Pages number first .. last - 1 hold nothing that is still seen."""

        for i in range(first, last):
            if self.pages[i] is not None:
                self.free.append(self.pages[i])
                self.pages[i] = None
                self.table[0, i] = -1


def serve_window(prompt_tokens=200, steps=150, window=64, sinks=4, width=256, page=16, pages=24, seed=0):
    """A prompt and then tokens one by one: outputs, tokens, layer, and how many pages were in use at most behind the prompt."""

    gen = torch.Generator(device="cuda").manual_seed(seed)
    layer = AttentionLayer(width, 4, 2, 64, 4096, seed=seed)
    cache, used = Cache(layer, pages, page), 0
    x = torch.randn(1, prompt_tokens + steps, width, generator=gen, device="cuda").bfloat16()
    q, k, v = layer.project(x[:, :prompt_tokens], None)
    append_tokens(k, v, cache.keys, cache.values, cache.slots(prompt_tokens))
    cache.length = prompt_tokens
    outs = [window_attention(q, k, v, window, sinks=sinks)]
    for i in range(prompt_tokens, prompt_tokens + steps):
        # what the window has left behind it, but for the sinks' pages
        cache.give_back(-(-sinks // page), max(0, cache.length - window + 1) // page)
        used = max(used, sum(p is not None for p in cache.pages))
        q, k, v = layer.project(x[:, i:i + 1], cache.lengths()[:, None].long())
        outs.append(window_tree_attention(q, k, v, cache.keys, cache.values, cache.table, cache.lengths(), window, sinks=sinks))
        append_tokens(k, v, cache.keys, cache.values, cache.slots(1))
        cache.length += 1
    return torch.cat(outs, 1), x, layer, used


def serve_evicting(prompt_tokens=200, steps=150, keep=96, room=32, sinks=4, recent=16, width=256, page=16, pages=40, seed=0):
    """The same with a cache that is thinned out to `keep` tokens whenever it has grown by `room`: outputs, and the cache's length
    ahead of every step."""

    gen = torch.Generator(device="cuda").manual_seed(seed)
    layer = AttentionLayer(width, 4, 2, 64, 4096, seed=seed)
    cache, lengths = Cache(layer, pages, page), []
    x = torch.randn(1, prompt_tokens + steps, width, generator=gen, device="cuda").bfloat16()
    q, k, v = layer.project(x[:, :prompt_tokens], None)
    out, weights = weighed_attention(q, k, v)
    slots = cache.slots(prompt_tokens)
    append_tokens(k, v, cache.keys, cache.values, slots)
    cache.weights[slots[0] // page, :, slots[0] % page] = weights[0]
    cache.length, outs = prompt_tokens, [out]
    for i in range(prompt_tokens, prompt_tokens + steps):
        if cache.length >= keep + room:
            old = list(cache.pages)
            fresh = [cache.free.pop() for _ in range(-(-keep // page))]
            new_table = torch.tensor([fresh], device="cuda", dtype=torch.int32)
            evict_tokens(cache.keys, cache.values, cache.weights, cache.table, cache.lengths(), new_table, keep, sinks=sinks, recent=recent)
            cache.free += old
            cache.pages, cache.length = fresh, keep
            cache.table.fill_(-1)
            cache.table[:, :len(fresh)] = new_table
        lengths.append(cache.length)
        # (a token's position goes on, whatever has left the cache)
        q, k, v = layer.project(x[:, i:i + 1], torch.tensor([[i]], device="cuda"))
        slots = cache.slots(1)
        outs.append(weighed_token_attention(q, k, v, cache.keys, cache.values, cache.weights, cache.table, cache.lengths(), slots))
        append_tokens(k, v, cache.keys, cache.values, slots)
        cache.length += 1
    return torch.cat(outs, 1), lengths


def main():
    loss, grads = training_step()
    print(f"training step: loss {loss.item():.4f}, {len(grads)} gradients, all finite: {all(torch.isfinite(g).all().item() for g in grads)}")
    got, tokens, layer, used = serve_window()
    q, k, v = layer.project(tokens, None)
    want = window_attention(q, k, v, 64, sinks=4)
    off = ((got - want).float().norm() / want.float().norm()).item()
    print(f"window: {tokens.shape[1]} tokens in up to {used} pages, off by {off:.1e} from one prompt of them all")
    out, lengths = serve_evicting()
    print(f"eviction: {out.shape[1]} tokens, a cache of up to {max(lengths[1:])} tokens, all finite: {torch.isfinite(out).all().item()}")


if __name__ == "__main__":
    main()
