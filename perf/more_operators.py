"""A KV cache held in 4 bits, and windows whose first tokens stay visible: what the operators compute, over which sizes,
and what one pass of each has to read, write and compute.

``append``: rows of the fused projection (q | k | v) of every request's new tokens; q and k get their RMS norm (q the
learned |temperature| too) and the rotary embedding of the token's position; q comes back, k and v go to the pages of
the request's cache in 4 bits; then the new tokens' keys and values are read back. ``read``: the last keys and values of
every request, read back from the 4-bit cache as bf16 rows. ``chunk``: attention of every request's new tokens over the
4-bit cache, causal, optionally with a sliding window and first tokens that stay visible, optionally with the layer's
output gate. ``sinks``: the same over a cache of bf16.

The 4-bit cache: 32 consecutive elements of a token's head are a group, x = m + s c with m the group's smallest element,
s = bf16((largest - smallest) / 15) and c = floor((x - m) / s + 1/2) in 0 .. 15. A pool is [pages, KV heads, page size /
16, 20 head dims] bytes: blocks of 16 tokens of a head, in each the codes of its 16 keys, those of its 16 values, the
(s, m) of the keys' groups and those of the values'. A row's codes are 32-bit words, word t * groups + g with elements
32 g + 8 t + e, e = 0 .. 7, element e in bits 4 (e // 2 + 4 (e % 2)) and up.

``run`` computes them with elementary torch operations in 32 bits where ``own`` is false (angles in 64), and calls the
package where it is true. ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
THETA = 10000.0


def listed():
    model = dict(heads=16, kv_heads=4, head_dim=128, half=False, rotary=128)  # the layer of the benchmark step
    free = dict(window=0, sinks=0)
    return [
        # one stream's next token: a launch's latency
        dict(name="append-1", op="append", streams=1, new=1, cached=877, ragged="", page=16, gate=False, mix=0, **model, **free),
        # the decode step of 256 streams
        dict(name="append-256x1", op="append", streams=256, new=1, cached=500, ragged="", page=16, gate=False, mix=0, **model, **free),
        # 256 prompts of up to 128 tokens prefilled at once
        dict(name="append-prompts", op="append", streams=256, new=128, cached=0, ragged="new", page=16, gate=False, mix=1,
             **model, **free),
        # one long prefix handed over to a cache of another kind
        dict(name="read-65536", op="read", streams=1, new=65536, cached=0, ragged="", page=64, gate=False, mix=0, **model, **free),
        # the tails of 64 ragged streams, two KV heads of 64, an odd page
        dict(name="read-ragged", op="read", streams=64, new=301, cached=129, ragged="both", page=48, gate=False, mix=2, heads=14,
             kv_heads=2, head_dim=64, half=True, rotary=32, **free),
        # one stream's next token over a short cache: latency
        dict(name="decode-1", op="chunk", streams=1, new=1, cached=877, ragged="", page=16, gate=True, mix=0, **model, **free),
        # the decode step of 256 streams at the end of a 1500-step generation
        dict(name="decode-256", op="chunk", streams=256, new=1, cached=1627, ragged="", page=16, gate=True, mix=0, **model, **free),
        # two streams deep into a long context: few rows over a long axis
        dict(name="decode-2-long", op="chunk", streams=2, new=1, cached=65000, ragged="", page=64, gate=True, mix=0, **model, **free),
        # chunked prefill: the next 512 tokens of four long prompts
        dict(name="chunk-4x512", op="chunk", streams=4, new=512, cached=8192, ragged="", page=32, gate=True, mix=0, **model, **free),
        # a serving batch: most streams decode, some bring a chunk, some nothing; a window with the first tokens kept
        dict(name="mixed-48", op="chunk", streams=48, new=384, cached=4096, ragged="mixed", page=16, gate=True, mix=4, window=1000,
             sinks=5, **model),
        # one long prompt of a model with windows, cache of bf16
        dict(name="sinks-prompt-8192", op="sinks", streams=1, new=8192, cached=0, ragged="", page=128, gate=True, mix=0, window=1024,
             sinks=4, **model),
        # endless streams: single tokens far behind their window's first tokens, cache of bf16
        dict(name="sinks-decode-64", op="sinks", streams=64, new=1, cached=16383, ragged="", page=16, gate=True, mix=0, window=1024,
             sinks=4, **model),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        heads, kv_heads = rng.choice([(16, 4), (8, 2), (8, 8), (14, 2), (16, 2), (6, 2), (4, 1)])
        head_dim = rng.choice([32, 64, 64, 96, 128, 128, 128])
        op = rng.choice(["append", "read", "chunk", "chunk", "chunk", "sinks"])
        attends = op in ("chunk", "sinks")
        windowed = op == "sinks" or (attends and rng.random() < 0.3)
        case = dict(op=op, streams=_log_int(rng, 1, 256), new=_log_int(rng, 1, 8192), cached=_log_int(rng, 1, 65000) - 1,
                    ragged=rng.choice(["", "new", "both", "mixed"]),
                    page=rng.choice([1, 7, 16, 24, 64, 128] if op == "sinks" else [16, 32, 48, 64, 128, 256]),
                    gate=attends and rng.random() < 0.5, mix=rng.randrange(1 << 20), heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, window=_log_int(rng, 1, 4096) if windowed else 0,
                    sinks=rng.choice([1, 4, _log_int(rng, 1, 300)]) if windowed else 0, half=rng.random() < 0.5,
                    rotary=rng.choice([head_dim, head_dim, head_dim // 2]))
        if attends and rng.random() < 0.4:  # decode batches
            case["new"] = rng.choice([1, 1, 2, 4])
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
    """Seconds of making and passing a case in its plain form, roughly: it works on requests padded to the longest."""
    new, keys = _lengths(case)
    rows = sum(keys) * case["kv_heads"] * case["head_dim"]
    if case["op"] in ("append", "read"):
        return rows * 4e-11 + sum(new) * case["heads"] * case["head_dim"] * 8e-11
    cells = len(new) * max(new) * max(keys) * case["heads"]
    padded = len(new) * max(keys) * case["kv_heads"] * case["head_dim"]
    return cells * (4 * case["head_dim"] / 5e13 + 4e-11) + padded * 1e-11 + rows * 2e-11


def _pairs(n, length, window, sinks):
    """(query, key) pairs that a request's new tokens see, and the keys that any of them sees."""
    pairs = 0
    for i in range(n):
        seen = length - n + i + 1
        pairs += min(seen, window + min(sinks, max(0, seen - window))) if window else seen
    if n == 0:
        return 0, 0
    below = max(0, length - n + 1 - window) if window else 0  # keys before the first token's window
    return pairs, length - below + min(sinks, below)


def work(case):
    new, keys = _lengths(case)
    heads, kv, hd, rows = case["heads"], case["kv_heads"], case["head_dim"], sum(new)
    four = kv * hd * 5 // 4  # a token's key and value in 4 bits
    if case["op"] == "append":  # the projection rows in; q, the cache rows, and the values they stand for out
        return {"bytes": rows * ((heads + 2 * kv) * hd * 2 + heads * hd * 2 + four + kv * hd * 4),
                "flops": rows * (heads + kv) * hd * 8 + rows * kv * hd * 16}
    if case["op"] == "read":
        return {"bytes": rows * (four + kv * hd * 4), "flops": rows * kv * hd * 4}
    pairs = cached = 0
    for n, length in zip(new, keys):
        p, c = _pairs(n, length, case["window"], case["sinks"])
        pairs, cached = pairs + p, cached + c
    moved = rows * heads * hd * 2 * 2 + cached * (four if case["op"] == "chunk" else kv * hd * 4)
    return {"bytes": moved + (rows * heads * 2 if case["gate"] else 0), "flops": 4 * pairs * heads * hd}


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

    state = dict(case=case, longest=max(keys), most=max(new), rows=rows, page_table=table.to(dev),
                 cache_seqlens=torch.tensor(keys, dtype=torch.int32, device=dev),
                 cu_seqlens_q=torch.tensor(starts, dtype=torch.int32, device=dev))
    if case["op"] == "sinks":
        state["k_cache"], state["v_cache"] = normal(total, page, kv, hd), normal(total, page, kv, hd)
    elif case["op"] == "append":
        state["kv_cache"] = torch.zeros(total, kv, page // 16, 20 * hd, device=dev, dtype=torch.uint8)
    else:
        state["kv_cache"] = _in_four_bits(normal(total, page, kv, hd), normal(total, page, kv, hd))
    if case["op"] == "append":
        # q | k | v | gate, as the layer's projection leaves it; what lies two deviations out is rare there
        state["proj"] = normal(rows, (heads + 2 * kv) * hd + heads).clamp_(-2, 2)
        state["temp"] = (1 + 0.1 * normal(heads)).to(torch.bfloat16)
    elif case["op"] != "read":
        state["q"] = normal(rows, heads, hd)
        state["gate"] = normal(rows, heads) if case["gate"] else None
    return state


def run(state):
    case = state["case"]
    if own:
        from __graft_entry__ import load_package

        ops = load_package().ops
        batch = (state["page_table"], state["cache_seqlens"], state["cu_seqlens_q"])
        if case["op"] == "append":
            q = ops.gqa_append_q4(state["proj"], state["kv_cache"], *batch, heads=case["heads"], kv_heads=case["kv_heads"],
                                  temp=state["temp"], eps=EPS, rope_theta=THETA, rotary_dim=case["rotary"],
                                  interleaved=not case["half"])
            return [q, *ops.kv_read_q4(state["kv_cache"], *batch, state["rows"])]
        if case["op"] == "read":
            return list(ops.kv_read_q4(state["kv_cache"], *batch, state["rows"]))
        more = dict(window=case["window"], sinks=case["sinks"], gate=state["gate"])
        if case["op"] == "sinks":
            return [ops.gqa_chunk(state["q"], state["k_cache"], state["v_cache"], *batch, **more)]
        return [ops.gqa_chunk_q4(state["q"], state["kv_cache"], *batch, max_new=state["most"], **more)]
    if case["op"] == "append":
        return _plain_append(state)
    if case["op"] == "read":
        request, _, position = _owner(state, state["rows"])
        return [x.to(torch.bfloat16) for x in _values(state, request, position)]
    return _plain_chunk(state)


# ------------------------------------------------------------------------------------------------ the 4-bit cache


def _codes(x):
    """Codes [..., hd / 32, 32] (int32) and pairs (s, m) [..., hd / 32, 2] (bf16) of bf16 rows [..., hd]."""
    x = x.float().unflatten(-1, (-1, 32))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((high - low) / 15).to(torch.bfloat16).float()
    c = torch.floor((x - low) / torch.where(s > 0, s, 1.0) + 0.5).clamp(0, 15)
    return torch.where(s > 0, c, 0.0).to(torch.int32), torch.cat([s, low], -1).to(torch.bfloat16)


def _bytes_of(codes):
    """Rows of hd / 2 bytes of codes [..., groups, 32]."""
    e = torch.arange(8, device=codes.device)
    words = codes.unflatten(-1, (4, 8)).transpose(-2, -3)  # [..., t, group, e]
    words = (words.long() << 4 * (e // 2 + 4 * (e % 2))).sum(-1).flatten(-2)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).view(torch.uint8)


def _parts(cache):
    """The four parts of a cache's blocks, as views: codes [pages, kv, blocks, 16, hd / 2], pairs [..., 16, hd / 8] bytes."""
    hd = cache.shape[-1] // 20
    at = [0, 8 * hd, 16 * hd, 18 * hd, 20 * hd]
    return [cache[..., a:z].unflatten(-1, (16, -1)) for a, z in zip(at, at[1:])]


def _in_four_bits(k, v):
    """A pool that holds keys and values [pages, page, kv, hd]."""
    pages, page, kv, hd = k.shape
    cache = torch.empty(pages, kv, page // 16, 20 * hd, device=k.device, dtype=torch.uint8)
    parts = _parts(cache)
    for i, x in enumerate((k, v)):
        codes, pairs = _codes(x.unflatten(1, (-1, 16)).permute(0, 3, 1, 2, 4))
        parts[i].copy_(_bytes_of(codes))
        parts[2 + i].copy_(pairs.flatten(-2).contiguous().view(torch.uint8))
    return cache


def _values(state, request, position):
    """Keys and values [*, kv, hd] (fp32) of key positions of requests."""
    page = state["case"]["page"]
    at = state["page_table"].long()[request, position // page].clamp(min=0), position % page // 16, position % 16
    parts = [x.transpose(1, 2).transpose(2, 3)[at] for x in _parts(state["kv_cache"])]  # [*, kv, bytes]
    found = []
    for codes, pairs in ((parts[0], parts[2]), (parts[1], parts[3])):
        words = codes.contiguous().view(torch.int32).unflatten(-1, (4, -1)).transpose(-1, -2)  # [*, kv, group, t]
        e = torch.arange(8, device=codes.device, dtype=torch.int32)
        c = ((words[..., None] >> 4 * (e // 2 + 4 * (e % 2))) & 15).flatten(-2).float()  # [*, kv, group, 32]
        s, m = pairs.contiguous().view(torch.bfloat16).float().unflatten(-1, (-1, 2)).unbind(-1)
        found.append((m[..., None] + s[..., None] * c).flatten(-2))
    return found


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
    inverse = THETA ** (-torch.arange(0, rot, 2, device=x.device, dtype=torch.float64) / rot)
    angle = (position.double()[:, None] * inverse)[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if case["half"]:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    x = torch.cat([turned, x[..., rot:]], -1).to(torch.bfloat16)
    k, v = x[:, heads:], proj[:, (heads + kv) * hd: (heads + 2 * kv) * hd].reshape(rows, kv, hd)
    where = state["page_table"].long()[request, position // page], position % page // 16, position % 16
    parts = [part.transpose(1, 2).transpose(2, 3) for part in _parts(state["kv_cache"])]
    (k_codes, k_pairs), (v_codes, v_pairs) = _codes(k), _codes(v)
    parts[0][where], parts[1][where] = _bytes_of(k_codes), _bytes_of(v_codes)
    parts[2][where], parts[3][where] = (p.flatten(-2).contiguous().view(torch.uint8) for p in (k_pairs, v_pairs))
    return [x[:, :heads].contiguous()] + [y.to(torch.bfloat16) for y in _values(state, request, position)]


def _plain_chunk(state):
    case, q = state["case"], state["q"]
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    rows, group, most, longest = q.shape[0], heads // kv, state["most"], state["longest"]
    request, index, position = _owner(state, rows)
    cu, lengths = state["cu_seqlens_q"].long(), state["cache_seqlens"].long()
    B = len(lengths)
    row = (cu[:-1, None] + torch.arange(most, device=q.device)).clamp(max=rows - 1)  # [B, most], padded
    at = lengths[:, None] - (cu[1:] - cu[:-1])[:, None] + torch.arange(most, device=q.device)
    key = torch.arange(longest, device=q.device)
    seen = (key[None, None, :] <= at[:, :, None]) & (key[None, None, :] < lengths[:, None, None])
    if case["window"]:
        seen = seen & ((key[None, None, :] > at[:, :, None] - case["window"]) | (key < case["sinks"]))
    every = torch.arange(B, device=q.device)[:, None]
    if case["op"] == "chunk":
        k, v = _values(state, every, key.expand(B, -1))  # [B, longest, kv, hd]
    else:
        pages = state["page_table"].long()[:, key // page].clamp(min=0)
        k, v = state["k_cache"][pages, key % page].float(), state["v_cache"][pages, key % page].float()
    part = q.float().unflatten(1, (kv, group))[row]  # [B, most, kv, group, hd]
    part = part.permute(0, 2, 3, 1, 4).reshape(B, kv, group * most, hd)
    s = (part @ k.permute(0, 2, 3, 1)).view(B, kv, group, most, longest) * hd ** -0.5
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = s.sum(-1)
    o = (s.view(B, kv, group * most, longest) @ v.transpose(1, 2)).view(B, kv, group, most, hd)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    out = o.permute(0, 3, 1, 2, 4)[request, index].flatten(1, 2)  # [rows, heads, hd]
    if state["gate"] is not None:
        out = out * (1.0 / (1.0 + torch.exp(-state["gate"].float())))[..., None]
    return [out.to(torch.bfloat16)]


# ------------------------------------------------------------------------------------------------ definition


def _places(hd):
    """Byte of a row of codes, and bit in it, of every element."""
    byte, bit = [], []
    for d in range(hd):
        group, t, e = d // 32, d % 32 // 8, d % 8
        nibble = e // 2 + 4 * (e % 2)
        byte.append(4 * (t * (hd // 32) + group) + nibble // 2)
        bit.append(4 * (nibble % 2))
    return torch.tensor(byte, device="cuda"), torch.tensor(bit, device="cuda")


def _read_exactly(cache, pages, offset, page):
    """Keys and values [n, kv, hd] in 64 bits of rows `offset` of `pages`."""
    hd = cache.shape[-1] // 20
    byte, bit = _places(hd)
    blocks = cache[pages, :, offset // 16]  # [n, kv, 20 hd]
    inside = (offset % 16)[:, None, None]
    group = torch.arange(hd, device="cuda") // 32
    found = []
    for part in range(2):
        c = blocks.gather(2, (part * 8 * hd + inside * (hd // 2) + byte).expand(-1, blocks.shape[1], -1))
        c = ((c.int() >> bit) & 15).double()
        start = (16 + 2 * part) * hd + inside * (hd // 8) + 4 * group
        raw = [blocks.gather(2, (start + i).expand(-1, blocks.shape[1], -1)).long() for i in range(4)]
        s, m = ((raw[2 * i] | raw[2 * i + 1] << 8).to(torch.int32).to(torch.int16).view(torch.bfloat16).double() for i in range(2))
        found.append(m + s * c)
    return found


def _stands_for(x):
    """The values that 4 bits keep of rows [n, kv, hd], in 64 bits."""
    g = x.to(torch.bfloat16).double().reshape(*x.shape[:-1], -1, 32)
    m = g.min(-1, keepdim=True).values
    s = ((g.max(-1, keepdim=True).values - m) / 15).to(torch.bfloat16).double()
    c = torch.where(s > 0, ((g - m) / s.clamp_min(1e-300) + 0.5).floor().clamp(max=15), torch.zeros_like(g))
    return (m + s * c).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    new, keys = _lengths(case)
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    table, rows = state["page_table"].cpu(), sum(new)
    if case["op"] in ("append", "read"):
        q_out = torch.empty(rows, heads, hd, device="cuda", dtype=torch.float64)
        k_out, v_out = (torch.empty(rows, kv, hd, device="cuda", dtype=torch.float64) for _ in range(2))
        rot, at = case["rotary"], 0
        # the rotation as a complex product: pair j turns by position * theta^(-2j / rot)
        pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
        first = pair.long() if case["half"] else 2 * pair.long()
        second = first + (rot // 2 if case["half"] else 1)
        for b, n in enumerate(new):
            if n == 0:
                continue
            p = torch.arange(keys[b] - n, keys[b])
            if case["op"] == "read":
                pages, offset = table[b, p // page].long().cuda(), (p % page).cuda()
                k_out[at:at + n], v_out[at:at + n] = _read_exactly(state["kv_cache"], pages, offset, page)
                at += n
                continue
            part = state["proj"][at:at + n].double()
            qk = part[:, : (heads + kv) * hd].unflatten(1, (heads + kv, hd))
            qk = qk / (qk.square().sum(-1, keepdim=True) / hd + EPS).sqrt()
            qk[:, :heads] *= state["temp"].double().abs().unsqueeze(-1)
            turn = torch.polar(torch.ones(n, rot // 2, device="cuda", dtype=torch.float64),
                               p.cuda().double()[:, None] * torch.exp(pair * (-2.0 * math.log(THETA) / rot)))
            z = torch.complex(qk[..., first], qk[..., second]) * turn[:, None]
            qk[..., first], qk[..., second] = z.real, z.imag
            q_out[at:at + n], k_out[at:at + n] = qk[:, :heads], _stands_for(qk[:, heads:])
            v_out[at:at + n] = _stands_for(part[:, (heads + kv) * hd: (heads + 2 * kv) * hd].unflatten(1, (kv, hd)))
            at += n
        return [q_out, k_out, v_out] if case["op"] == "append" else [k_out, v_out]
    out = torch.zeros(rows, heads, hd, device="cuda", dtype=torch.float64)
    at = 0
    for b, (n, length) in enumerate(zip(new, keys)):
        if n == 0:
            continue
        p = torch.arange(length)
        pages, offset = table[b, p // page].long().cuda(), (p % page).cuda()
        row = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = p.cuda()[None] > row
        if case["window"]:
            hidden |= (p.cuda()[None] <= row - case["window"]) & (p.cuda()[None] >= case["sinks"])
        if case["op"] == "chunk":
            k_all, v_all = _read_exactly(state["kv_cache"], pages, offset, page)
        else:
            k_all, v_all = state["k_cache"][pages, offset].double(), state["v_cache"][pages, offset].double()
        for h in range(kv):
            for g in range(h * heads // kv, (h + 1) * heads // kv):
                s = state["q"][at:at + n, g].double() @ k_all[:, h].t() / math.sqrt(hd)
                s.masked_fill_(hidden, float("-inf"))
                s -= s.max(-1, keepdim=True).values
                s.exp_()
                out[at:at + n, g] = (s @ v_all[:, h]) / s.sum(-1, keepdim=True)
        if state["gate"] is not None:
            out[at:at + n] *= torch.sigmoid(state["gate"][at:at + n].double()).unsqueeze(-1)
        at += n
    return [out]
