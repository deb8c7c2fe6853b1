"""Workloads of attention layers whose memory of the past is bounded: by a sliding window, or by eviction from the cache.

A case is a dict of plain values; ``kind`` says which operator it goes through:

  prompt   window_attention ([batch, time]) or window_attention_varlen (``lengths``): a token sees the ``window`` last tokens,
           itself among them, and the first ``sinks`` of its sequence; no gradients
  train    the same with the gradients of q, k and v
  tree     window_tree_attention: ``drafted`` tokens of each of ``batch`` sequences over a paged cache of up to ``context`` tokens
           a sequence (each between a quarter of it and all of it), of which the window and the sinks are read; one drafted
           token is plain decoding, ``branches`` says that several form a tree and not a chain
  weigh    weighed_attention or weighed_attention_varlen: causal attention, and the weight that every token got from all
           queries, summed over the heads of a group
  step     weighed_token_attention: attention of ``tokens`` new tokens a sequence over a paged cache; what weight each cached
           token got is added to its weight so far times ``decay``.  With a decay of 1 a new period of observation begins with
           every pass, so that it can be repeated: the weights start from 0
  evict    evict_tokens: of every sequence and key head the ``keep`` tokens of the largest weights are copied to other pages,
           the first ``sinks`` and the last ``recent`` of a sequence in any case

``dtype`` is the type of queries, keys and values, which are N(0, 1); weights are in 32 bits.
"""

import math

import torch

own = False  # False: the plain forms below; True: the framework's operators

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ELEMENT = 2


def listed():
    return [
        # the prefill configuration of the benchmark (8 prompts of 4096 tokens, 16 heads), a window of a quarter
        dict(name="prompt_b8_t4096_w1024", kind="prompt", batch=8, time=4096, heads=16, kv_heads=4, dim=128, window=1024, sinks=4,
             dtype="bf16"),
        # one long document of no round length, one shared key head, a wide window
        dict(name="prompt_b1_t16381_w4096", kind="prompt", batch=1, time=16381, heads=8, kv_heads=1, dim=128, window=4096, sinks=128,
             dtype="fp16"),
        # a training step
        dict(name="train_b4_t2048_w512", kind="train", batch=4, time=2048, heads=16, kv_heads=4, dim=128, window=512, sinks=16,
             dtype="bf16"),
        # packed documents of odd lengths, smaller heads, none shared, a window of no round size and no sinks
        dict(name="train_packed_d64_w333", kind="train", lengths="1021,513,77,1500,1,389,2047,640", heads=8, kv_heads=8, dim=64,
             window=333, sinks=0, dtype="fp16"),
        # plain decoding of a full batch whose contexts are longer than the window
        dict(name="token_b64_c16384_w4096", kind="tree", batch=64, drafted=1, branches=False, context=16384, heads=32, kv_heads=8,
             dim=128, page=64, window=4096, sinks=4, dtype="bf16"),
        # trees of drafted tokens, an odd window, small pages
        dict(name="tree24_b8_c9000_w1000", kind="tree", batch=8, drafted=24, branches=True, context=9000, heads=16, kv_heads=4,
             dim=128, page=16, window=1000, sinks=64, dtype="fp16"),
        # prompts whose cache will be thinned out
        dict(name="weigh_b4_t4096", kind="weigh", batch=4, time=4096, heads=16, kv_heads=4, dim=128, dtype="bf16"),
        # many short requests, packed
        dict(name="weigh_packed_short", kind="weigh", lengths="1,2,17,33,64,65,90,127,128,129,150,200,211,255,256,300,7,48,77,181",
             heads=16, kv_heads=2, dim=64, dtype="fp16"),
        # a decoding step of a full batch
        dict(name="step_b64_c8192", kind="step", batch=64, tokens=1, context=8192, heads=32, kv_heads=8, dim=128, page=64, decay=1.0,
             dtype="bf16"),
        # one user, a short context: nothing but latency
        dict(name="step_b1_c301", kind="step", batch=1, tokens=1, context=301, heads=16, kv_heads=2, dim=128, page=16, decay=0.0,
             dtype="fp16"),
        # caches of long prompts are thinned out to a quarter
        dict(name="evict_b8_n16384_k4096", kind="evict", batch=8, context=16384, keep=4096, sinks=4, recent=256, kv_heads=8, dim=128,
             page=64, dtype="bf16"),
        # caches that have grown by some pages since the last time, pages of no round size
        dict(name="evict_b24_n1203_k1024", kind="evict", batch=24, context=1203, keep=1024, sinks=0, recent=100, kv_heads=4, dim=96,
             page=24, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "train", "train", "tree", "tree", "weigh", "step", "step", "evict"])
    dtype, page = rng.choice(["bf16", "fp16"]), rng.choice([16, 24, 32, 64, 128])
    kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 96, 128])
    heads = kv_heads * group
    sinks = rng.choice([0, 0, 1, 4, 16, 64, 128, _log(rng, 1, 300)])
    if kind in ("prompt", "train", "weigh"):
        heads = min(heads, 16)
        kv_heads = heads // group if heads % group == 0 else heads
        case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
        if kind != "weigh":
            case.update(window=_log(rng, 1, 4096), sinks=sinks)
        most = int(5e7 if kind == "train" else 5e8) // heads  # (query, key) pairs of a head, were there no window
        if rng.random() < 0.5:
            batch = _log(rng, 1, 16)
            case.update(batch=batch, time=_log(rng, 1, min(8192, math.isqrt(most // batch))))
        else:
            count = _log(rng, 1, 48)
            longest = min(4096, math.isqrt(most // count))
            case.update(lengths=",".join(str(_log(rng, 1, longest)) for _ in range(count)))
        return case
    batch = _log(rng, 1, 64)
    heads = min(heads, 32)
    kv_heads = heads // group if heads % group == 0 else heads
    most = 64 * 8192 * 8 * 128 // (batch * max(heads // 4, kv_heads) * dim)  # tokens a sequence of the largest cache
    if kind == "evict":
        context = _log(rng, 1, max(1, min(20000, most // 4)))
        keep = _log(rng, 1, context + 10)
        sinks = min(sinks, keep)
        return dict(kind=kind, batch=batch, context=context, keep=keep, sinks=sinks, recent=rng.randint(0, keep - sinks),
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    context = _log(rng, 1, max(1, min(20000, most)))
    case = dict(kind=kind, batch=batch, context=context, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if kind == "tree":
        drafted = rng.choice([1, 1, _log(rng, 2, 64)])
        case.update(drafted=drafted, branches=drafted > 1 and rng.random() < 0.7, window=_log(rng, 1, 8192), sinks=sinks)
    else:
        case.update(tokens=rng.choice([1, 1, 1, 2, 5]), decay=rng.choice([0.0, 1.0]))
    return case


def _lengths(case):
    if "lengths" in case:
        return [int(x) for x in case["lengths"].split(",")]
    return [case["time"]] * case["batch"]


def _contexts(case):
    """Cached tokens of every sequence: spread between a quarter of the largest and all of it (caches to be thinned out: between
    all of it and seven eighths)."""

    n, top = case["batch"], case["context"]
    less = top // 8 if case["kind"] == "evict" else 3 * top // 4
    return [max(1, top - less * ((5 * i) % n) // n) for i in range(n)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dim, kv_heads, kind = TYPES[case["dtype"]], case["dim"], case["kv_heads"], case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    state = {"case": dict(case)}
    if kind in ("prompt", "train", "weigh"):
        lengths, heads = _lengths(case), case["heads"]
        lead = (1, sum(lengths)) if "lengths" in case else (case["batch"], case["time"])
        state.update(q=normal(*lead, heads, dim), k=normal(*lead, kv_heads, dim), v=normal(*lead, kv_heads, dim))
        bounds = [0]
        for n in lengths:
            bounds.append(bounds[-1] + n)
        state["bounds"] = tuple(bounds)
        if kind == "train":
            state["do"] = normal(*lead, heads, dim)
            for name in "qkv":
                state[name].requires_grad_(True)
        return state
    batch, page, contexts = case["batch"], case["page"], _contexts(case)
    room = case["tokens"] if kind == "step" else 0  # the new tokens' places
    need = [-(-(n + room) // page) for n in contexts]
    kept = -(-case["keep"] // page) if kind == "evict" else 0
    pages = sum(need) + batch * kept + 5
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.zeros(batch, max(need), device="cuda", dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    state.update(k_pages=normal(pages, page, kv_heads, dim), v_pages=normal(pages, page, kv_heads, dim), page_table=table,
                 lengths=torch.tensor(contexts, device="cuda", dtype=torch.int32))
    if kind != "tree":
        # what tokens have got so far: few of them most of it
        state["weight_pages"] = torch.empty(pages, kv_heads, page, device="cuda").exponential_(1.0, generator=gen)
    if kind == "evict":
        state["new_table"] = order[at:at + batch * kept].view(batch, kept).contiguous()
        return state
    n = case["drafted"] if kind == "tree" else case["tokens"]
    state.update(q=normal(batch, n, case["heads"], dim), k=normal(batch, n, kv_heads, dim), v=normal(batch, n, kv_heads, dim))
    if kind == "step":
        place = state["lengths"].long()[:, None] + torch.arange(n, device="cuda")
        state["slots"] = table.long().gather(1, place // page) * page + place % page
        return state
    state.update(mask=None, depths=None)
    if case["branches"]:
        # every drafted token continues an earlier one (the first continues the context): it sees its ancestors
        parent = (torch.rand(batch, n, generator=gen, device="cuda") * torch.arange(n, device="cuda")).long()
        mask = torch.eye(n, device="cuda", dtype=torch.bool).repeat(batch, 1, 1)
        which = torch.arange(batch, device="cuda")
        for i in range(1, n):
            mask[:, i] |= mask[which, parent[:, i]]
        state.update(mask=mask, depths=mask.sum(-1, dtype=torch.int32) - 1)
    return state


# ---- plain forms: elementary operations in 32 bits, rounded once -----------------------------------------------


def _weights(scores, seen):
    """Softmax over the keys that are seen; zeros where none is."""

    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _sequences(bounds):
    """Where the rows of packed sequences are: number of the sequence, place in it."""

    row = torch.arange(bounds[-1], device="cuda")
    starts = torch.tensor(bounds, device="cuda")
    sequence = torch.searchsorted(starts, row, right=True) - 1
    return sequence, row - starts[sequence]


def _padded(x, n, longest, where):
    """[sequences, heads, longest, dim] in 32 bits, zeros behind a sequence's end."""

    out = x.new_zeros((n, longest, *x.shape[2:]), dtype=torch.float32)
    out[where] = x.detach().flatten(0, 1).float()
    return out.transpose(1, 2)


def _plain_attention(s):
    case, bounds = s["case"], s["bounds"]
    group, scale = case["heads"] // case["kv_heads"], case["dim"] ** -0.5
    n, longest = len(bounds) - 1, max(b - a for a, b in zip(bounds, bounds[1:]))
    where = _sequences(bounds)

    def packed(x, like):
        return x.transpose(1, 2)[where].to(like.dtype).view(like.shape)

    q, k, v = (_padded(s[name], n, longest, where) for name in "qkv")
    _, kv_heads, _, dim = k.shape
    q = q.view(n, kv_heads, group, longest, dim)
    i, j = torch.arange(longest, device="cuda")[:, None], torch.arange(longest, device="cuda")
    seen = j <= i
    if case["kind"] != "weigh":
        seen = seen & ((i - j < case["window"]) | (j < case["sinks"]))
    p = _weights(q @ k[:, :, None].transpose(-1, -2) * scale, seen)
    o = p @ v[:, :, None]
    out = packed(o.flatten(1, 2), s["q"])
    if case["kind"] == "weigh":
        there = i < torch.tensor([b - a for a, b in zip(bounds, bounds[1:])], device="cuda")[:, None, None, None, None]
        got = (p * there).sum((2, 3)).transpose(1, 2)[where]
        return out, got.view(*s["k"].shape[:3])
    if case["kind"] == "prompt":
        return out
    do = _padded(s["do"], n, longest, where).view(q.shape)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = p * (do @ v[:, :, None].transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * scale
    dq, dk = ds @ k[:, :, None], (ds.transpose(-1, -2) @ q).sum(2)
    return out, packed(dq.flatten(1, 2), s["q"]), packed(dk, s["k"]), packed(dv, s["v"])


def _plain_paged(s):
    case = s["case"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    batch, n, heads, dim = q.shape
    kv_heads, page = k.shape[2], s["k_pages"].shape[1]
    table, length = s["page_table"].long(), s["lengths"].long()
    cached = [s[name][table].flatten(1, 2).float() for name in ("k_pages", "v_pages")]
    k, v = (torch.cat(pair, 1).transpose(1, 2) for pair in zip(cached, (k, v)))
    reach = cached[0].shape[1]
    t, i = torch.arange(reach, device=q.device), torch.arange(n, device=q.device)
    context = (t < length[:, None])[:, None].expand(batch, n, reach)
    if case["kind"] == "tree" and s["mask"] is not None:
        mask, depth = s["mask"], s["depths"].long()
    else:
        mask, depth = (i <= i[:, None]).expand(batch, n, n), i.expand(batch, n)
    if case["kind"] == "tree":
        at = length[:, None] + depth  # places of the drafted tokens
        context = context & ((at[:, :, None] - t < case["window"]) | (t < case["sinks"]))
        mask = mask & ((depth[:, :, None] - depth[:, None] < case["window"]) | (at[:, None] < case["sinks"]))
    q = q.view(batch, n, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    p = _weights(q @ k[:, :, None].transpose(-1, -2) * dim ** -0.5, torch.cat([context, mask], -1)[:, None, None])
    out = (p @ v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(s["q"].shape).to(s["q"].dtype)
    if case["kind"] == "tree":
        return out
    got, weights, page_of = p.sum((2, 3)).transpose(1, 2), s["weight_pages"], t // page
    if case["decay"] == 1.0:
        weights.zero_()
    there = t < length[:, None]
    where = (table[:, page_of][there], slice(None), (t % page).expand(batch, reach)[there])
    weights[where] = weights[where] * case["decay"] + got[:, :reach][there]
    weights[s["slots"] // page, :, s["slots"] % page] = got[:, reach:]
    return out, weights


def _plain_evict(s):
    case, keep = s["case"], s["case"]["keep"]
    table, to, length = s["page_table"].long(), s["new_table"].long(), s["lengths"].long()[:, None, None]
    (_, page, kv_heads, dim), batch = s["k_pages"].shape, table.shape[0]
    weights = s["weight_pages"][table].transpose(1, 2).flatten(2)  # [batch, head, token]
    t = torch.arange(weights.shape[2], device="cuda")
    stays = (t < case["sinks"]) | (t >= length - case["recent"])
    weights = torch.where(t >= length, -math.inf, torch.where(stays, math.inf, weights))
    kept = weights.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    there = torch.arange(kept.shape[2], device="cuda") < length  # (all of a sequence that is no longer)
    there = there.expand(kept.shape)
    b = torch.arange(batch, device="cuda")[:, None, None]
    head = torch.arange(kv_heads, device="cuda")[:, None].expand(kept.shape)[there]
    x = torch.arange(kept.shape[2], device="cuda")
    from_page, from_place = table[b, kept // page][there], (kept % page)[there]
    to_page, to_place = to[b, x // page].expand(kept.shape)[there], (x % page).expand(kept.shape)[there]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[to_page, to_place, head] = pages[from_page, from_place, head]
    s["weight_pages"][to_page, head, to_place] = s["weight_pages"][from_page, head, from_place]
    return s["k_pages"], s["v_pages"], s["weight_pages"], s["lengths"].clamp(max=keep)


def run(state):
    s, case, kind = state, state["case"], state["case"]["kind"]
    if not own:
        return {"prompt": _plain_attention, "train": _plain_attention, "weigh": _plain_attention, "tree": _plain_paged,
                "step": _plain_paged, "evict": _plain_evict}[kind](s)
    if kind == "tree":
        from gdn2_sm120_b200.window import window_tree_attention

        return window_tree_attention(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], case["window"],
                                     s["mask"], s["depths"], sinks=case["sinks"])
    if kind == "step":
        from gdn2_sm120_b200.eviction import weighed_token_attention

        if case["decay"] == 1.0:
            s["weight_pages"].zero_()
        out = weighed_token_attention(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["weight_pages"], s["page_table"],
                                      s["lengths"], s["slots"], decay=case["decay"])
        return out, s["weight_pages"]
    if kind == "evict":
        from gdn2_sm120_b200.eviction import evict_tokens

        lengths = evict_tokens(s["k_pages"], s["v_pages"], s["weight_pages"], s["page_table"], s["lengths"], s["new_table"],
                               case["keep"], sinks=case["sinks"], recent=case["recent"])
        return s["k_pages"], s["v_pages"], s["weight_pages"], lengths
    if kind == "weigh":
        from gdn2_sm120_b200.eviction import weighed_attention, weighed_attention_varlen

        if "lengths" in case:
            return weighed_attention_varlen(s["q"], s["k"], s["v"], s["bounds"])
        return weighed_attention(s["q"], s["k"], s["v"])
    from gdn2_sm120_b200.window import window_attention, window_attention_varlen

    if "lengths" in case:
        out = window_attention_varlen(s["q"], s["k"], s["v"], s["bounds"], case["window"], sinks=case["sinks"])
    else:
        out = window_attention(s["q"], s["k"], s["v"], case["window"], sinks=case["sinks"])
    if kind == "prompt":
        return out
    return out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])


# ---- the definitions in 64 bits, a sequence and a head at a time -----------------------------------------------


def _probabilities(q, k, seen):
    s = (q @ k.T / math.sqrt(k.shape[1])).masked_fill(~seen, -math.inf)
    return torch.softmax(s, -1).nan_to_num(0.0)


def _exact_attention(s):
    case, bounds = s["case"], s["bounds"]
    group, kind = case["heads"] // case["kv_heads"], case["kind"]
    flat = {name: s[name].detach().flatten(0, 1) for name in ("q", "k", "v", "do") if name in s}
    out = torch.zeros(flat["q"].shape, device="cuda", dtype=torch.float64)
    got = torch.zeros(flat["k"].shape[:2], device="cuda", dtype=torch.float64)
    grads = {name: torch.zeros(flat[name].shape, device="cuda", dtype=torch.float64) for name in "qkv"} if kind == "train" else None
    for lo, hi in zip(bounds, bounds[1:]):
        for h in range(case["heads"]):
            q, k, v = flat["q"][lo:hi, h].double(), flat["k"][lo:hi, h // group].double(), flat["v"][lo:hi, h // group].double()
            for r in range(0, hi - lo, 4096):
                e = min(hi - lo, r + 4096)
                i, j = torch.arange(r, e, device="cuda")[:, None], torch.arange(e, device="cuda")
                seen = j <= i
                if kind != "weigh":
                    seen = seen & ((j > i - case["window"]) | (j < case["sinks"]))
                leaves = [x.clone().requires_grad_(grads is not None) for x in (q[r:e], k[:e], v[:e])]
                p = _probabilities(leaves[0], leaves[1], seen)
                y = p @ leaves[2]
                out[lo + r:lo + e, h] = y.detach()
                if kind == "weigh":
                    got[lo:lo + e, h // group] += p.sum(0)
                if grads is not None:
                    dq, dk, dv = torch.autograd.grad(y, leaves, flat["do"][lo + r:lo + e, h].double())
                    grads["q"][lo + r:lo + e, h] = dq
                    grads["k"][lo:lo + e, h // group] += dk
                    grads["v"][lo:lo + e, h // group] += dv
    out = out.view(s["q"].shape)
    if kind == "weigh":
        return out, got.view(s["k"].shape[:3])
    return out if grads is None else (out, *(grads[name].view(s[name].shape) for name in "qkv"))


def _exact_paged(s):
    case = s["case"]
    batch, n, heads, _ = s["q"].shape
    kv_heads, page = s["k"].shape[2], s["k_pages"].shape[1]
    group = heads // kv_heads
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    weights = s["weight_pages"].double() * (case["decay"] != 1.0) if case["kind"] == "step" else None
    i = torch.arange(n, device="cuda")
    for b in range(batch):
        length = int(s["lengths"][b])
        t = torch.arange(length, device="cuda")
        pages, places = s["page_table"][b, t // page].long(), t % page
        k, v = (torch.cat([s[name + "_pages"][pages, places], s[name][b]]).double() for name in "kv")
        place = torch.cat([t, length + i])
        tail, at = i <= i[:, None], length + i
        if case["kind"] == "tree" and s["mask"] is not None:
            tail, at = s["mask"][b], length + s["depths"][b].long()
            place = torch.cat([t, at])
        seen = torch.cat([torch.ones(n, length, device="cuda", dtype=torch.bool), tail], 1)
        if case["kind"] == "tree":
            seen = seen & ((place > at[:, None] - case["window"]) | (place < case["sinks"]))
        for g in range(kv_heads):
            q = s["q"][b, :, g * group:(g + 1) * group].double().flatten(0, 1)
            p = _probabilities(q, k[:, g], seen.repeat_interleave(group, 0))
            out[b, :, g * group:(g + 1) * group] = (p @ v[:, g]).view(n, group, -1)
            if weights is not None:
                got = p.sum(0)
                weights[pages, g, places] = weights[pages, g, places] * case["decay"] + got[:length]
                weights[s["slots"][b] // page, g, s["slots"][b] % page] = got[length:]
    return out if weights is None else (out, weights)


def exact(case, seed):
    if case["kind"] == "evict":
        return None  # nothing but copies
    s = prepare(case, seed)
    return (_exact_paged if case["kind"] in ("tree", "step") else _exact_attention)(s)


def work(case):
    kind, dim, kv_heads = case["kind"], case["dim"], case["kv_heads"]

    def pairs(n):  # of a sequence's queries and the keys that they see
        if kind == "weigh":
            return n * (n + 1) // 2
        window, sinks = min(case["window"], n), min(case["sinks"], n)
        behind = n - window  # queries that do not see the first token for their window
        return window * (window + 1) // 2 + behind * window + sum(min(x, sinks) for x in range(1, behind + 1))

    if kind in ("prompt", "train", "weigh"):
        lengths, heads = _lengths(case), case["heads"]
        total = heads * sum(pairs(n) for n in lengths)
        q, kv = sum(lengths) * heads * dim * ELEMENT, sum(lengths) * kv_heads * dim * ELEMENT
        if kind == "train":
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * dim * total}
        return {"bytes": 2 * q + 2 * kv + (4 * sum(lengths) * kv_heads if kind == "weigh" else 0), "flops": 4 * dim * total}
    contexts = _contexts(case)
    if kind == "evict":
        kept = kv_heads * sum(min(n, case["keep"]) for n in contexts)
        return {"bytes": 2 * kept * (2 * dim * ELEMENT) + 4 * (kv_heads * sum(contexts) + kept), "flops": 0}
    n, heads = case["drafted" if kind == "tree" else "tokens"], case["heads"]
    rows = case["batch"] * n
    if kind == "tree":  # what the first drafted token sees, which all the others nearly see too
        contexts = [min(x, case["window"] - 1) + max(0, min(case["sinks"], x - case["window"] + 1)) for x in contexts]
    seen = sum(contexts) + rows
    return {"bytes": 2 * seen * kv_heads * dim * ELEMENT + 2 * rows * heads * dim * ELEMENT + (4 * seen * kv_heads if kind == "step" else 0),
            "flops": 4 * dim * heads * n * sum(x + n for x in contexts)}
