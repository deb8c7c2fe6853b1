"""A full-attention layer beside a Gated DeltaNet-2 layer: one training step, then serving with drafted trees.

    python examples/attention_layer.py

``AttentionLayer`` runs the attention operators the way a stack of both kinds of layers does:

  training   rotary positions -> causal attention over packed sequences -> gradients
  prompts    the same without gradients; keys and values go into the pages of a cache
  drafts     rotary positions -> attention of a drafted tree over the cache; the accepted tokens are appended

``serve`` drafts a few trees, accepts a path of each and returns the layer's outputs for all accepted tokens: they are those
of one prompt that holds them all.
"""

from __future__ import annotations

import pathlib
import sys

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))

from gdn2_sm120_b200 import chunk_gdn2
from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen
from gdn2_sm120_b200.paged import append_tokens, tree_attention
from gdn2_sm120_b200.rotary import apply_rotary, rotary_tables


class AttentionLayer:
    """Projections, rotary positions, attention; ``width`` channels a token."""

    def __init__(self, width, heads, kv_heads, dim, positions, device="cuda", dtype=torch.bfloat16, seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.w_in = torch.randn(width, (heads + 2 * kv_heads) * dim, generator=gen, device=device, dtype=dtype) * width ** -0.5
        self.w_out = torch.randn(heads * dim, width, generator=gen, device=device, dtype=dtype) * (heads * dim) ** -0.5
        self.cos, self.sin = rotary_tables(positions, dim // 2, device=device)   # half of the channels turn

    def project(self, x, positions):
        """q, k, v of tokens [B, T, width]: views of one product, q and k turned."""

        parts = (x @ self.w_in).split([n * self.dim for n in (self.heads, self.kv_heads, self.kv_heads)], -1)
        q, k, v = (part.unflatten(-1, (-1, self.dim)) for part in parts)
        q, k = apply_rotary(q, k, self.cos, self.sin, positions, layout="interleaved")
        return q, k, v

    def train(self, x, cu_seqlens):
        """Packed sequences [1, total, width]; a token's position is its number in its sequence."""

        positions = torch.cat([torch.arange(b - a, device=x.device) for a, b in zip(cu_seqlens, cu_seqlens[1:])])
        q, k, v = self.project(x, positions)
        return causal_attention_varlen(q, k, v, cu_seqlens).flatten(-2) @ self.w_out

    def prompt(self, x, cache, slots):
        """A prompt [1, T, width]; its keys and values go to the cache's slots."""

        q, k, v = self.project(x, None)
        append_tokens(k, v, *cache, slots)
        return causal_attention(q, k, v).flatten(-2) @ self.w_out

    def drafts(self, x, depth, mask, cache, page_table, lengths):
        """A drafted tree [B, N, width]: a token's position is the context's length and its depth.  Returns the outputs
        and the keys and values, of which the caller appends what it accepts."""

        q, k, v = self.project(x, lengths[:, None] + depth)
        return tree_attention(q, k, v, *cache, page_table, lengths, mask).flatten(-2) @ self.w_out, k, v


def training_step(lengths=(70, 1, 200), width=256, seed=0):
    """Gated DeltaNet-2, then attention, over packed sequences: the loss and every gradient."""

    device, heads = "cuda", 2
    gen = torch.Generator(device=device).manual_seed(seed)
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    layer = AttentionLayer(width, 4, 2, 64, max(lengths))
    q, k, v, beta, w = (torch.randn(1, bounds[-1], heads, 128, generator=gen, device=device).bfloat16() for _ in range(5))
    g = -torch.rand(1, bounds[-1], heads, 128, generator=gen, device=device) * 0.1
    q, k = (torch.nn.functional.normalize(x.float(), dim=-1).bfloat16() for x in (q, k))
    leaves = [x.requires_grad_(True) for x in (q, k, v, g, beta.sigmoid(), w.sigmoid(), layer.w_in, layer.w_out)]
    # (one recurrence over all rows: chunk_gdn2_varlen keeps the sequences apart)
    mixed, _ = chunk_gdn2(*leaves[:6])
    out = layer.train(mixed.flatten(-2), tuple(bounds))
    loss = out.float().square().mean()
    return loss.detach(), torch.autograd.grad(loss, leaves)


def serve(prompt_tokens=100, rounds=4, width=256, page=16, seed=0):
    """Outputs of all accepted tokens of one sequence, and those tokens."""

    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    layer = AttentionLayer(width, 4, 2, 64, 4096, seed=seed)
    pages = (prompt_tokens + 3 * rounds) // page + 2
    cache = tuple(torch.zeros(pages, page, layer.kv_heads, layer.dim, device=device, dtype=torch.bfloat16) for _ in range(2))
    page_table = torch.randperm(pages, generator=gen, device=device).int()[None]

    def slots(first, count):
        at = torch.arange(first, first + count, device=device)
        return page_table[0, at // page].long() * page + at % page

    x = torch.randn(1, prompt_tokens, width, generator=gen, device=device).bfloat16()
    outs, tokens, length = [layer.prompt(x, cache, slots(0, prompt_tokens)[None])], [x], prompt_tokens
    # two branches from the context, 0 -> 1 -> 2 and 3 -> 4
    parent, depth = [-1, 0, 1, -1, 3], torch.tensor([0, 1, 2, 0, 1], device=device)
    mask = torch.eye(5, device=device, dtype=torch.bool)
    for i, j in enumerate(parent):
        if j >= 0:
            mask[i] |= mask[j]
    for step in range(rounds):
        draft = torch.randn(1, 5, width, generator=gen, device=device).bfloat16()
        out, k, v = layer.drafts(draft, depth, mask, cache, page_table, torch.tensor([length], device=device, dtype=torch.int32))
        path = ([0, 1, 2], [3, 4], [0], [3])[step % 4]       # what verification accepts
        to = torch.full((1, 5), -1, device=device)           # the others stay outside the cache
        to[0, path] = slots(length, len(path))
        append_tokens(k, v, *cache, to)
        outs.append(out[:, path])
        tokens.append(draft[:, path])
        length += len(path)
    return torch.cat(outs, 1), torch.cat(tokens, 1), layer


def main():
    loss, grads = training_step()
    print(f"training step: loss {loss.item():.4f}, {len(grads)} gradients, all finite: {all(torch.isfinite(g).all().item() for g in grads)}")
    got, tokens, layer = serve()
    q, k, v = layer.project(tokens, None)
    want = causal_attention(q, k, v).flatten(-2) @ layer.w_out
    off = ((got - want).float().norm() / want.float().norm()).item()
    print(f"serving: {tokens.shape[1]} tokens, drafted ones off by {off:.1e} from one prompt of them all")


if __name__ == "__main__":
    main()
