"""Workloads of the operators of an attention layer that stands between Gated DeltaNet-2 layers.

A case is a dict of plain values; ``kind`` says which operator it goes through:

  rotary   apply_rotary: q [B, T, heads, dim] and k [B, T, kv_heads, dim] turned by the angles of their positions;
           ``rotated`` channels of a head, ``layout`` half or interleaved; ``grad``: the gradients too
  append   append_tokens: keys and values of ``tokens`` tokens written to their slots of a paged cache; about
           ``skipped`` of a hundred have no slot (rejected drafts)
  prompt   causal_attention ([batch, time]) or causal_attention_varlen (``lengths``) without gradients
  train    the same with the gradients of q, k and v
  tree     tree_attention: ``drafted`` tokens of each of ``batch`` sequences over a cache of up to ``context`` tokens
           a sequence (each between a quarter of it and all of it), pages of ``page`` tokens in no order;
           one drafted token is plain decoding

``dtype`` is the type of every tensor but the rotary tables (fp32).  Inputs are N(0, 1).
"""

import math

import torch

own = False  # False: the plain forms below; True: the framework's operators

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ELEMENT = 2


def listed():
    return [
        # one decoding step of a full batch: nothing but latency
        dict(name="rotary_step_b64", kind="rotary", batch=64, time=1, heads=32, kv_heads=8, dim=128, rotated=128,
             layout="half", table=32768, grad=False, dtype="bf16"),
        # a training step's rotation, half of the channels, with the gradients
        dict(name="rotary_train_b2_t8192", kind="rotary", batch=2, time=8192, heads=32, kv_heads=8, dim=128, rotated=64,
             layout="interleaved", table=8192, grad=True, dtype="fp16"),
        # the tokens of one decoding step go into the cache
        dict(name="append_step_64", kind="append", tokens=64, kv_heads=8, dim=128, page=64, skipped=0, dtype="bf16"),
        # prompts and accepted drafts go into the cache
        dict(name="append_prompt_16411", kind="append", tokens=16411, kv_heads=8, dim=128, page=16, skipped=10, dtype="bf16"),
        # many short requests, packed
        dict(name="prompt_packed_short", kind="prompt", lengths="1,2,17,33,64,65,90,127,128,129,150,200,211,255,256,300,7,48,77,181",
             heads=16, kv_heads=4, dim=128, dtype="bf16"),
        # the prefill configuration of the benchmark (8 prompts of 4096 tokens, 16 heads), four heads a group
        dict(name="prompt_b8_t4096", kind="prompt", batch=8, time=4096, heads=16, kv_heads=4, dim=128, dtype="bf16"),
        # one long document of no round length, one shared key head
        dict(name="prompt_b1_t16381", kind="prompt", batch=1, time=16381, heads=8, kv_heads=1, dim=128, dtype="fp16"),
        # a training step
        dict(name="train_b4_t2048", kind="train", batch=4, time=2048, heads=16, kv_heads=4, dim=128, dtype="bf16"),
        # packed documents of odd lengths, smaller heads, none shared
        dict(name="train_packed_d64", kind="train", lengths="1021,513,77,1500,1,389,2047,640", heads=8, kv_heads=8, dim=64,
             dtype="fp16"),
        # plain decoding of a full batch
        dict(name="token_b64_c8192", kind="tree", batch=64, drafted=1, context=8192, heads=32, kv_heads=8, dim=128, page=64,
             dtype="bf16"),
        # trees of 48 drafted tokens over long contexts
        dict(name="tree48_b8_c16000", kind="tree", batch=8, drafted=48, context=16000, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16"),
        # one user, a small tree, a short context: nothing but latency
        dict(name="tree7_b1_c301", kind="tree", batch=1, drafted=7, context=301, heads=16, kv_heads=2, dim=128, page=16,
             dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "prompt", "prompt", "train", "train", "tree", "tree"])
    dtype = rng.choice(["bf16", "fp16"])
    kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 96, 128])
    heads = kv_heads * group
    if kind == "rotary":
        batch = _log(rng, 1, 64)
        time = _log(rng, 1, max(1, min(8192, 2 * 8192 * 40 * 128 // (batch * (heads + kv_heads) * dim))))
        return dict(kind=kind, batch=batch, time=time, heads=heads, kv_heads=kv_heads, dim=dim,
                    rotated=rng.choice([dim, dim // 2]), layout=rng.choice(["half", "interleaved"]), table=32768,
                    grad=rng.choice([True, False]), dtype=dtype)
    if kind == "append":
        return dict(kind=kind, tokens=_log(rng, 1, 16000), kv_heads=kv_heads, dim=dim, page=rng.choice([16, 24, 32, 64, 128]),
                    skipped=rng.choice([0, 0, 10, 50]), dtype=dtype)
    if kind in ("prompt", "train"):
        heads = min(heads, 16)
        kv_heads = heads // group if heads % group == 0 else heads
        case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
        most = int(8e7 if kind == "train" else 5e8) // heads  # (query, key) pairs of a head
        if rng.random() < 0.5:
            batch = _log(rng, 1, 16)
            case.update(batch=batch, time=_log(rng, 1, min(8192, math.isqrt(most // batch))))
        else:
            count = _log(rng, 1, 48)
            longest = min(4096, math.isqrt(most // count))
            case.update(lengths=",".join(str(_log(rng, 1, longest)) for _ in range(count)))
        return case
    batch, drafted = _log(rng, 1, 64), rng.choice([1, 1, _log(rng, 2, 64)])
    heads = min(heads, 32)
    kv_heads = heads // group if heads % group == 0 else heads
    most = 64 * 8192 * 8 * 128 // (batch * max(heads // 4, kv_heads) * dim)  # no more cache than the largest listed case reads
    return dict(kind=kind, batch=batch, drafted=drafted, context=_log(rng, 1, max(1, min(20000, most))), heads=heads,
                kv_heads=kv_heads, dim=dim, page=rng.choice([16, 24, 32, 64, 128]), dtype=dtype)


def _lengths(case):
    if "lengths" in case:
        return [int(x) for x in case["lengths"].split(",")]
    return [case["time"]] * case["batch"]


def _contexts(case):
    """Cached tokens of every sequence: spread between a quarter of the largest and all of it."""

    n, top = case["batch"], case["context"]
    return [max(1, top - (3 * top // 4) * ((5 * i) % n) // n) for i in range(n)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dim, kv_heads = TYPES[case["dtype"]], case["dim"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    state = {"case": dict(case)}
    if case["kind"] == "rotary":
        batch, time, heads = case["batch"], case["time"], case["heads"]
        pairs = case["rotated"] // 2
        speed = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
        angle = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * speed
        state.update(q=normal(batch, time, heads, dim), k=normal(batch, time, kv_heads, dim),
                     cos=angle.cos().float(), sin=angle.sin().float())
        first = torch.randint(0, case["table"] - time + 1, (batch, 1), generator=gen, device="cuda")
        state["positions"] = first + torch.arange(time, device="cuda")
        if case["grad"]:
            state.update(dq=normal(batch, time, heads, dim), dk=normal(batch, time, kv_heads, dim))
            state["q"].requires_grad_(True)
            state["k"].requires_grad_(True)
    elif case["kind"] == "append":
        tokens, page = case["tokens"], case["page"]
        pages = tokens // page + 9
        state.update(k=normal(tokens, kv_heads, dim), v=normal(tokens, kv_heads, dim),
                     k_pages=normal(pages, page, kv_heads, dim), v_pages=normal(pages, page, kv_heads, dim))
        order = torch.randperm(pages, generator=gen, device="cuda")  # whole pages in no order
        at = torch.arange(tokens, device="cuda")
        slots = order[at // page] * page + at % page
        skip = torch.randint(0, 100, (tokens,), generator=gen, device="cuda") < case["skipped"]
        state["slots"] = torch.where(skip, -1, slots)
    elif case["kind"] in ("prompt", "train"):
        lengths, heads = _lengths(case), case["heads"]
        lead = (1, sum(lengths)) if "lengths" in case else (case["batch"], case["time"])
        state.update(q=normal(*lead, heads, dim), k=normal(*lead, kv_heads, dim), v=normal(*lead, kv_heads, dim))
        bounds = [0]
        for n in lengths:
            bounds.append(bounds[-1] + n)
        state["bounds"] = tuple(bounds)
        row = torch.arange(bounds[-1], device="cuda")
        starts = torch.tensor(bounds, device="cuda")
        state["sequence"] = torch.searchsorted(starts, row, right=True) - 1
        state["offset"] = row - starts[state["sequence"]]
        if case["kind"] == "train":
            state["do"] = normal(*lead, heads, dim)
            for name in "qkv":
                state[name].requires_grad_(True)
    else:
        batch, drafted, page, heads = case["batch"], case["drafted"], case["page"], case["heads"]
        contexts = _contexts(case)
        columns = -(-max(contexts) // page)
        pages = sum(-(-n // page) for n in contexts) + 5
        state.update(q=normal(batch, drafted, heads, dim), k=normal(batch, drafted, kv_heads, dim),
                     v=normal(batch, drafted, kv_heads, dim), k_pages=normal(pages, page, kv_heads, dim),
                     v_pages=normal(pages, page, kv_heads, dim))
        order = torch.randperm(pages, generator=gen, device="cuda").int()
        table = torch.zeros(batch, columns, device="cuda", dtype=torch.int32)
        at = 0
        for i, n in enumerate(contexts):
            need = -(-n // page)
            table[i, :need] = order[at:at + need]
            at += need
        state.update(page_table=table, lengths=torch.tensor(contexts, device="cuda", dtype=torch.int32), mask=None)
        if drafted > 1:
            # every drafted token continues an earlier one (the first continues the context): it sees its ancestors
            parent = (torch.rand(batch, drafted, generator=gen, device="cuda") * torch.arange(drafted, device="cuda")).long()
            mask = torch.eye(drafted, device="cuda", dtype=torch.bool).repeat(batch, 1, 1)
            which = torch.arange(batch, device="cuda")
            for i in range(1, drafted):
                mask[:, i] |= mask[which, parent[:, i]]
            state["mask"] = mask
    return state


# ---- plain forms: elementary operations in 32 bits, rounded once -----------------------------------------------


def _turn(x, cos, sin, rotated, layout):
    x = x.float()
    turned, rest = x[..., :rotated], x[..., rotated:]
    if layout == "half":
        a, b = turned[..., :rotated // 2], turned[..., rotated // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _plain_rotary(s):
    case, dtype = s["case"], s["q"].dtype
    how = (case["rotated"], case["layout"])
    cos, sin = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
    out = [_turn(s[name].detach(), cos, sin, *how).to(dtype) for name in ("q", "k")]
    if case["grad"]:  # the transposed rotation
        out += [_turn(s[name], cos, -sin, *how).to(dtype) for name in ("dq", "dk")]
    return out


def _plain_append(s):
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    s["k_pages"].view(-1, *s["k"].shape[1:])[at] = s["k"][keep]
    s["v_pages"].view(-1, *s["v"].shape[1:])[at] = s["v"][keep]
    return s["k_pages"], s["v_pages"]


def _weights(scores, seen):
    """Softmax over the keys that are seen; zeros where none is."""

    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _padded(s, x, longest):
    """[sequences, heads, longest, dim] in 32 bits, zeros behind a sequence's end."""

    out = x.new_zeros((len(s["bounds"]) - 1, longest, *x.shape[2:]), dtype=torch.float32)
    out[s["sequence"], s["offset"]] = x.detach().flatten(0, 1).float()
    return out.transpose(1, 2)


def _packed(s, x, like):
    return x.transpose(1, 2)[s["sequence"], s["offset"]].to(like.dtype).view(like.shape)


def _plain_attention(s):
    case, group = s["case"], s["case"]["heads"] // s["case"]["kv_heads"]
    scale, longest = case["dim"] ** -0.5, max(b - a for a, b in zip(s["bounds"], s["bounds"][1:]))
    q, k, v = (_padded(s, s[name], longest) for name in "qkv")
    n, kv_heads, _, dim = k.shape
    q = q.view(n, kv_heads, group, longest, dim)
    seen = torch.ones(longest, longest, device=q.device, dtype=torch.bool).tril()
    p = _weights(q @ k[:, :, None].transpose(-1, -2) * scale, seen)
    o = p @ v[:, :, None]
    out = _packed(s, o.flatten(1, 2), s["q"])
    if case["kind"] == "prompt":
        return out
    do = _padded(s, s["do"], longest).view(q.shape)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = p * (do @ v[:, :, None].transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * scale
    dq, dk = ds @ k[:, :, None], (ds.transpose(-1, -2) @ q).sum(2)
    return out, _packed(s, dq.flatten(1, 2), s["q"]), _packed(s, dk, s["k"]), _packed(s, dv, s["v"])


def _plain_tree(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    batch, drafted, heads, dim = q.shape
    kv_heads = k.shape[2]
    table = s["page_table"].long()
    cached = [s[name][table].flatten(1, 2).float() for name in ("k_pages", "v_pages")]
    k, v = (torch.cat(pair, 1).transpose(1, 2) for pair in zip(cached, (k, v)))
    reach = cached[0].shape[1]
    context = torch.arange(reach, device=q.device) < s["lengths"][:, None]
    mask = s["mask"] if s["mask"] is not None else torch.ones(batch, 1, 1, device=q.device, dtype=torch.bool)
    seen = torch.cat([context[:, None].expand(batch, drafted, reach), mask], -1)
    q = q.view(batch, drafted, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    p = _weights(q @ k[:, :, None].transpose(-1, -2) * dim ** -0.5, seen[:, None, None])
    o = p @ v[:, :, None]
    return o.permute(0, 3, 1, 2, 4).reshape(s["q"].shape).to(s["q"].dtype)


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "prompt": _plain_attention, "train": _plain_attention,
                "tree": _plain_tree}[kind](s)
    if kind == "rotary":
        from gdn2_sm120_b200.rotary import apply_rotary

        q, k = apply_rotary(s["q"], s["k"], s["cos"], s["sin"], s["positions"], layout=s["case"]["layout"])
        if not s["case"]["grad"]:
            return [q, k]
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return [q.detach(), k.detach(), dq, dk]
    if kind == "append":
        from gdn2_sm120_b200.paged import append_tokens

        return append_tokens(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"])
    if kind == "tree":
        from gdn2_sm120_b200.paged import tree_attention

        return tree_attention(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["mask"])
    from gdn2_sm120_b200.attention import causal_attention, causal_attention_varlen

    if "lengths" in s["case"]:
        out = causal_attention_varlen(s["q"], s["k"], s["v"], s["bounds"])
    else:
        out = causal_attention(s["q"], s["k"], s["v"])
    if kind == "prompt":
        return out
    return out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------


def _exact_rotary(s):
    case = s["case"]
    pairs = case["rotated"] // 2
    i = torch.arange(pairs, device="cuda")
    first, second = (i, i + pairs) if case["layout"] == "half" else (2 * i, 2 * i + 1)
    phase = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, :, None]

    def turned(x, by):
        y = x.detach().double().clone()
        z = torch.complex(y[..., first], y[..., second]) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = [turned(s["q"], phase), turned(s["k"], phase)]
    if case["grad"]:
        out += [turned(s["dq"], phase.conj()), turned(s["dk"], phase.conj())]
    return out


def _exact_append(s):
    k, v = s["k_pages"].double().clone(), s["v_pages"].double().clone()
    page = k.shape[1]
    token = torch.nonzero(s["slots"] >= 0).flatten()
    where = s["slots"][token]
    k[where // page, where % page] = s["k"][token].double()
    v[where // page, where % page] = s["v"][token].double()
    return k, v


def _rows(q, k, v, seen):
    """Output of query rows: q [rows, dim], k and v [keys, dim]; `seen` [rows, keys]."""

    logits = (q @ k.T) / math.sqrt(q.shape[1])
    logits[~seen] = -math.inf
    norm = torch.logsumexp(logits, 1, keepdim=True)
    return torch.exp(logits - norm.clamp_min(-1e300)) @ v


def _exact_attention(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    flat = {name: s[name].detach().flatten(0, 1) for name in ("q", "k", "v", "do") if name in s}
    out = torch.empty(flat["q"].shape, device="cuda", dtype=torch.float64)
    grads = {name: torch.zeros(flat[name].shape, device="cuda", dtype=torch.float64) for name in "qkv"} if "do" in flat else None
    for lo, hi in zip(s["bounds"], s["bounds"][1:]):
        for h in range(case["heads"]):
            q, k, v = flat["q"][lo:hi, h].double(), flat["k"][lo:hi, h // group].double(), flat["v"][lo:hi, h // group].double()
            for r in range(0, hi - lo, 4096):
                e = min(hi - lo, r + 4096)
                seen = torch.arange(e, device="cuda") <= torch.arange(r, e, device="cuda")[:, None]
                leaves = [x.clone().requires_grad_(grads is not None) for x in (q[r:e], k[:e], v[:e])]
                y = _rows(*leaves, seen)
                out[lo + r:lo + e, h] = y.detach()
                if grads is not None:
                    dq, dk, dv = torch.autograd.grad(y, leaves, flat["do"][lo + r:lo + e, h].double())
                    grads["q"][lo + r:lo + e, h] = dq
                    grads["k"][lo:lo + e, h // group] += dk
                    grads["v"][lo:lo + e, h // group] += dv
    out = out.view(s["q"].shape)
    return out if grads is None else (out, *(grads[name].view(s[name].shape) for name in "qkv"))


def _exact_tree(s):
    batch, drafted, heads, _ = s["q"].shape
    kv_heads, page = s["k"].shape[2], s["k_pages"].shape[1]
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    for b in range(batch):
        n = int(s["lengths"][b])
        at = torch.arange(n, device="cuda")
        at = s["page_table"][b, at // page].long() * page + at % page
        k, v = (torch.cat([s[name + "_pages"].flatten(0, 1)[at], s[name][b]]).double() for name in "kv")
        tail = s["mask"][b] if s["mask"] is not None else torch.ones(drafted, drafted, device="cuda", dtype=torch.bool).tril()
        seen = torch.cat([torch.ones(drafted, n, device="cuda", dtype=torch.bool), tail], 1)
        for h in range(heads):
            g = h // (heads // kv_heads)
            out[b, :, h] = _rows(s["q"][b, :, h].double(), k[:, g], v[:, g], seen)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "prompt": _exact_attention, "train": _exact_attention,
            "tree": _exact_tree}[case["kind"]](s)


def work(case):
    kind, dim, kv_heads = case["kind"], case["dim"], case["kv_heads"]
    if kind == "rotary":
        tokens, per = case["batch"] * case["time"], (case["heads"] + kv_heads) * dim
        passes = 2 if case["grad"] else 1
        angles = min(case["table"], tokens) * case["rotated"] * 4
        return {"bytes": passes * (2 * tokens * per * ELEMENT) + angles + 8 * tokens,
                "flops": passes * 3 * tokens * (case["heads"] + kv_heads) * case["rotated"]}
    if kind == "append":
        kept = case["tokens"] * (100 - case["skipped"]) // 100
        return {"bytes": 4 * kept * kv_heads * dim * ELEMENT + 8 * case["tokens"], "flops": 0}
    if kind in ("prompt", "train"):
        lengths, heads = _lengths(case), case["heads"]
        pairs = heads * sum(n * (n + 1) // 2 for n in lengths)
        q, kv = sum(lengths) * heads * dim * ELEMENT, sum(lengths) * kv_heads * dim * ELEMENT
        if kind == "prompt":
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * dim * pairs}
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * dim * pairs}
    contexts, drafted, heads = _contexts(case), case["drafted"], case["heads"]
    rows = case["batch"] * drafted
    return {"bytes": 2 * (sum(contexts) + rows) * kv_heads * dim * ELEMENT + 2 * rows * heads * dim * ELEMENT,
            "flops": 4 * dim * heads * drafted * sum(n + drafted for n in contexts)}
