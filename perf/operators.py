"""The operators of the global-attention layers over a paged KV cache: what they compute, over which sizes, and what
one pass of each has to read, write and compute.

``append``: rows of the fused projection (q | k | v) of every request's new tokens; q and k get their RMS norm (q the
learned |temperature| too) and the rotary embedding of the token's position; q comes back, k and v go to the pages of
the request's cache. ``chunk``: attention of every request's new tokens (one, a few, a whole prompt, or none) over
the request's pages, causal, optionally within a sliding window, optionally with the layer's output gate.

``run`` computes them with elementary torch operations in 32 bits where ``own`` is false, and calls the package where
it is true. ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
THETA = 10000.0


def listed():
    model = dict(heads=16, kv_heads=4, head_dim=128, window=0, half=False, rotary=128)  # the layer of the benchmark step
    return [
        # one stream's next token: a launch's latency
        dict(name="append-1", op="append", streams=1, new=1, cached=877, ragged="", page=1, gate=False, mix=0, **model),
        # the decode step of 256 streams
        dict(name="append-256x1", op="append", streams=256, new=1, cached=500, ragged="", page=16, gate=False, mix=0,
             **model),
        # 256 prompts of up to 128 tokens prefilled at once
        dict(name="append-prompts", op="append", streams=256, new=128, cached=0, ragged="new", page=16, gate=False,
             mix=1, **model),
        # ragged chunks behind ragged caches, an odd page, seven query heads to a KV head, half of each head rotated
        dict(name="append-odd", op="append", streams=37, new=301, cached=129, ragged="both", page=24, gate=False, mix=2,
             heads=14, kv_heads=2, head_dim=64, window=0, half=True, rotary=32),
        # one stream's next token over a short cache: latency
        dict(name="decode-1", op="chunk", streams=1, new=1, cached=877, ragged="", page=1, gate=True, mix=0, **model),
        # the decode step of 256 streams at the end of a 1500-step generation
        dict(name="decode-256", op="chunk", streams=256, new=1, cached=1627, ragged="", page=16, gate=True, mix=0,
             **model),
        # two streams deep into a long context: few rows over a long axis
        dict(name="decode-2-long", op="chunk", streams=2, new=1, cached=65000, ragged="", page=64, gate=True, mix=0,
             **model),
        # 256 prompts of up to 128 tokens prefilled at once
        dict(name="prompts-256", op="chunk", streams=256, new=128, cached=0, ragged="new", page=16, gate=True, mix=3,
             **model),
        # chunked prefill: the next 512 tokens of four long prompts
        dict(name="chunk-4x512", op="chunk", streams=4, new=512, cached=8192, ragged="", page=32, gate=True, mix=0,
             **model),
        # one long prompt
        dict(name="prompt-8192", op="chunk", streams=1, new=8192, cached=0, ragged="", page=128, gate=True, mix=0,
             **model),
        # a serving batch: most streams decode, some bring a chunk, some nothing
        dict(name="mixed-48", op="chunk", streams=48, new=384, cached=4096, ragged="mixed", page=16, gate=True, mix=4,
             **model),
        # sliding window, head dim 64, seven query heads to a KV head, odd page and lengths
        dict(name="window-odd", op="chunk", streams=9, new=777, cached=3001, ragged="both", page=24, gate=False, mix=5,
             heads=14, kv_heads=2, head_dim=64, window=512, half=False, rotary=64),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        heads, kv_heads = rng.choice([(16, 4), (8, 2), (8, 8), (14, 2), (16, 2), (6, 2), (4, 1)])
        head_dim = rng.choice([32, 64, 64, 96, 128, 128, 128])
        op = rng.choice(["append", "chunk", "chunk", "chunk"])
        case = dict(op=op, streams=_log_int(rng, 1, 256), new=_log_int(rng, 1, 8192), cached=_log_int(rng, 1, 65000) - 1,
                    ragged=rng.choice(["", "new", "both", "mixed"]), page=rng.choice([1, 7, 16, 24, 32, 64, 128, 256]),
                    gate=op == "chunk" and rng.random() < 0.5, mix=rng.randrange(1 << 20), heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim,
                    window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]) if op == "chunk" else 0,
                    half=rng.random() < 0.5, rotary=rng.choice([head_dim, head_dim, head_dim // 2]))
        new, keys = _lengths(case)
        if sum(new) and _cost(case) <= top:
            return case


def _lengths(case):
    """New tokens and keys (the new ones included) of every request."""
    rng = random.Random(case["mix"])
    new, keys = [], []
    for _ in range(case["streams"]):
        n, c = case["new"], case["cached"]
        if case["ragged"] in ("new", "both"):
            n = rng.randint(1, n)
        if case["ragged"] == "both":
            c = rng.randint(0, c)
        if case["ragged"] == "mixed":
            kind = rng.random()
            n = 1 if kind < 0.7 else 0 if kind < 0.75 else rng.randint(1, n)
            c = rng.randint(0, c)
        new.append(n)
        keys.append(n + c)
    return new, keys


def _cost(case):
    """Seconds of the plain form, roughly: it works on requests padded to the longest."""
    new, keys = _lengths(case)
    cells = len(new) * max(new) * max(keys) * case["heads"]
    rows = len(new) * max(keys) * case["kv_heads"] * case["head_dim"]
    if case["op"] == "append":
        return sum(keys) * case["kv_heads"] * case["head_dim"] * 4e-12 + sum(new) * case["heads"] * case["head_dim"] * 4e-11
    return cells * (4 * case["head_dim"] / 5e13 + 4e-11) + rows * 1e-11


def _pairs(n, length, window):
    """(query, key) pairs that a request's new tokens see, and the keys that any of them sees."""
    pairs = 0
    for i in range(n):
        seen = length - n + i + 1
        pairs += min(seen, window) if window else seen
    first = length - n + 1
    return pairs, (length if not window else length - max(0, first - window)) if n else 0


def work(case):
    new, keys = _lengths(case)
    heads, kv, hd, rows = case["heads"], case["kv_heads"], case["head_dim"], sum(new)
    if case["op"] == "append":  # the projection rows in; q and the new cache rows out
        width = (heads + 2 * kv) * hd
        return {"bytes": rows * width * 2 * 2, "flops": rows * (heads + kv) * hd * 8}
    pairs = cached = 0
    for n, length in zip(new, keys):
        p, c = _pairs(n, length, case["window"])
        pairs, cached = pairs + p, cached + c
    moved = rows * heads * hd * 2 * 2 + cached * kv * hd * 2 * 2 + (rows * heads * 2 if case["gate"] else 0)
    return {"bytes": moved, "flops": 4 * pairs * heads * hd}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    new, keys = _lengths(case)
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    pages = [-(-k // page) for k in keys]
    width = max(max(pages), 1)
    total = sum(pages) + 3
    order = torch.randperm(total, generator=gen, device=dev).to(torch.int32).cpu()
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    at = 0
    for b, count in enumerate(pages):
        table[b, :count] = order[at:at + count]
        at += count
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = starts[-1]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.bfloat16)

    state = dict(case=case, longest=max(keys), most=max(new), page_table=table.to(dev),
                 cache_seqlens=torch.tensor(keys, dtype=torch.int32, device=dev),
                 cu_seqlens_q=torch.tensor(starts, dtype=torch.int32, device=dev),
                 k_cache=normal(total, page, kv, hd), v_cache=normal(total, page, kv, hd))
    if case["op"] == "append":
        state["proj"] = normal(rows, (heads + 2 * kv) * hd + heads)  # q | k | v | gate, as the layer's projection leaves it
        state["temp"] = (1 + 0.1 * normal(heads)).to(torch.bfloat16)
    else:
        state["q"] = normal(rows, heads, hd)
        state["gate"] = normal(rows, heads) if case["gate"] else None
    return state


def run(state):
    case = state["case"]
    if own:
        from __graft_entry__ import load_package

        ops = load_package().ops
        paged = (state["k_cache"], state["v_cache"], state["page_table"], state["cache_seqlens"], state["cu_seqlens_q"])
        if case["op"] == "append":
            q = ops.gqa_append(state["proj"], *paged, heads=case["heads"], kv_heads=case["kv_heads"], temp=state["temp"],
                               eps=EPS, rope_theta=THETA, rotary_dim=case["rotary"], interleaved=not case["half"])
            return [q, state["k_cache"], state["v_cache"]]
        return [ops.gqa_chunk(state["q"], *paged, window=case["window"], gate=state["gate"])]
    return _plain_append(state) if case["op"] == "append" else _plain_chunk(state)


# ------------------------------------------------------------------------------------------------ plain forms


def _owner(state, rows):
    """Request, index among the request's new tokens and key position of every row."""
    cu = state["cu_seqlens_q"].long()
    token = torch.arange(rows, device=cu.device)
    request = torch.bucketize(token, cu[1:], right=True)
    index = token - cu[request]
    position = state["cache_seqlens"].long()[request] - (cu[request + 1] - cu[request]) + index
    return request, index, position


def _plain_append(state):
    case, proj = state["case"], state["proj"]
    heads, kv, hd, page, rot = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["rotary"]
    rows = proj.shape[0]
    request, _, position = _owner(state, rows)
    x = proj[:, : (heads + kv) * hd].reshape(rows, heads + kv, hd).float()
    x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))
    x[:, :heads] = x[:, :heads] * state["temp"].float().abs()[None, :, None]
    inverse = THETA ** (-torch.arange(0, rot, 2, device=x.device, dtype=torch.float32) / rot)
    angle = (position.float()[:, None] * inverse)[:, None, :]
    cos, sin = torch.cos(angle), torch.sin(angle)
    if case["half"]:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    x = torch.cat([turned, x[..., rot:]], -1).to(torch.bfloat16)
    where = state["page_table"].long()[request, position // page], position % page
    state["k_cache"][where] = x[:, heads:]
    state["v_cache"][where] = proj[:, (heads + kv) * hd: (heads + 2 * kv) * hd].reshape(rows, kv, hd)
    return [x[:, :heads].contiguous(), state["k_cache"], state["v_cache"]]


def _plain_chunk(state):
    case, q = state["case"], state["q"]
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    rows, group, most, longest = q.shape[0], heads // kv, state["most"], state["longest"]
    request, index, position = _owner(state, rows)
    cu, lengths = state["cu_seqlens_q"].long(), state["cache_seqlens"].long()
    row = (cu[:-1, None] + torch.arange(most, device=q.device)).clamp(max=rows - 1)  # [B, most], padded
    at = lengths[:, None] - (cu[1:] - cu[:-1])[:, None] + torch.arange(most, device=q.device)
    key = torch.arange(longest, device=q.device)
    pages = state["page_table"].long()[:, key // page].clamp(min=0)  # [B, longest]
    seen = (key[None, None, :] <= at[:, :, None]) & (key[None, None, :] < lengths[:, None, None])
    if case["window"]:
        seen = seen & (key[None, None, :] > at[:, :, None] - case["window"])
    out = torch.empty(rows, heads, hd, device=q.device, dtype=torch.float32)
    for h in range(kv):
        k = state["k_cache"][pages, key % page, h].float()  # [B, longest, hd]
        v = state["v_cache"][pages, key % page, h].float()
        part = q[:, h * group:(h + 1) * group].float()[row]  # [B, most, group, hd]
        part = part.transpose(1, 2).reshape(len(lengths), group * most, hd)
        s = torch.bmm(part, k.transpose(1, 2)).view(len(lengths), group, most, longest) * hd ** -0.5
        s = torch.where(seen[:, None], s, float("-inf"))
        top = s.amax(-1, keepdim=True)
        s = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
        total = s.sum(-1)
        o = torch.bmm(s.view(len(lengths), group * most, longest), v).view(len(lengths), group, most, hd)
        o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
        out[:, h * group:(h + 1) * group] = o[request, :, index]
    if state["gate"] is not None:
        out = out * (1.0 / (1.0 + torch.exp(-state["gate"].float())))[..., None]
    return [out.to(torch.bfloat16)]


# ------------------------------------------------------------------------------------------------ definition


def exact(case, seed):
    state = prepare(case, seed)
    new, keys = _lengths(case)
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    table = state["page_table"].cpu()
    if case["op"] == "append":
        rot, rows = case["rotary"], sum(new)
        q_out = torch.empty(rows, heads, hd, device="cuda", dtype=torch.float64)
        k_cache, v_cache = state["k_cache"].double(), state["v_cache"].double()
        # the rotation as a complex product: pair j turns by position * theta^(-2j / rot)
        pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
        first = pair.long() if case["half"] else 2 * pair.long()
        second = first + (rot // 2 if case["half"] else 1)
        at = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            p = torch.arange(keys[b] - n, keys[b])
            part = state["proj"][at:at + n].double()
            qk = part[:, : (heads + kv) * hd].unflatten(1, (heads + kv, hd))
            qk = qk / (qk.square().sum(-1, keepdim=True) / hd + EPS).sqrt()
            qk[:, :heads] *= state["temp"].double().abs().unsqueeze(-1)
            turn = torch.polar(torch.ones(n, rot // 2, device="cuda", dtype=torch.float64),
                               p.cuda().double()[:, None] * torch.exp(pair * (-2.0 * math.log(THETA) / rot)))
            z = torch.complex(qk[..., first], qk[..., second]) * turn[:, None]
            qk[..., first], qk[..., second] = z.real, z.imag
            pages, offset = table[b, p // page].long().cuda(), (p % page).cuda()
            q_out[at:at + n] = qk[:, :heads]
            k_cache[pages, offset] = qk[:, heads:]
            v_cache[pages, offset] = part[:, (heads + kv) * hd: (heads + 2 * kv) * hd].unflatten(1, (kv, hd))
            at += n
        return [q_out, k_cache, v_cache]
    out = torch.zeros(sum(new), heads, hd, device="cuda", dtype=torch.float64)
    at = 0
    for b, (n, length) in enumerate(zip(new, keys)):
        if n == 0:
            continue
        p = torch.arange(length)
        pages, offset = table[b, p // page].long().cuda(), (p % page).cuda()
        rows = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = p.cuda()[None] > rows
        if case["window"]:
            hidden |= p.cuda()[None] <= rows - case["window"]
        for h in range(kv):
            k, v = state["k_cache"][pages, offset, h].double(), state["v_cache"][pages, offset, h].double()
            for g in range(h * heads // kv, (h + 1) * heads // kv):
                s = state["q"][at:at + n, g].double() @ k.t() / math.sqrt(hd)
                s.masked_fill_(hidden, float("-inf"))
                s -= s.max(-1, keepdim=True).values
                s.exp_()
                out[at:at + n, g] = (s @ v) / s.sum(-1, keepdim=True)
        if state["gate"] is not None:
            out[at:at + n] *= torch.sigmoid(state["gate"][at:at + n].double()).unsqueeze(-1)
        at += n
    return [out]
