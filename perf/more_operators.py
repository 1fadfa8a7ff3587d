"""The operators of a key/value cache held in 4 bits, as their users call them.

  append    ``ops.qk_norm_rope_write_4bit``: per-head norm and rotation of q and k, k and v into 4-bit pages
  expand    ``ops.expand_pages_4bit``: the values of 4-bit pages, into pages of their own
  attend    ``ops.paged_attention_4bit``: attention of single tokens and of portions over 4-bit pages

Where ``own`` is false, ``run`` computes the same from elementary operations.

The cache: for every token, kv head and group of 32 neighbouring channels a step s and a least value m (bfloat16) and 32 codes c of 4 bits,
value = m + s c.  m is the largest bfloat16 not above the group's least value, s the smallest not below (largest - m) / 15, c = (x - m) / s
rounded, halves to even.  Pools are [pages, heads, page, width]: codes in bytes (width D / 2), steps (width D / 16: s and m of each group).
The 16-bit word r * D / 32 + g of a row of codes holds channels 32 g + 4 r to 32 g + 4 r + 3, the first in its lowest bits.
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GROUP = 32
EPS = 1e-6


def _append(name, tokens, heads, kv_heads, dim, dtype="bf16", page=16, norm=True, rotary=None):
    return dict(name=name, op="append", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, norm=norm, rotary=dim if rotary is None else rotary)


def _expand(name, seqs, keys, kv_heads, dim, dtype="bf16", page=16):
    return dict(name=name, op="expand", seqs=seqs, keys=keys, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page)


def _attend(name, seqs, keys, heads, kv_heads, dim, dtype="bf16", page=16, tokens=1, window=0, least=0.5):
    return dict(name=name, op="attend", seqs=seqs, keys=keys, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, tokens=tokens, window=window, least=least)


def listed():
    return [
        # the token of one conversation: latency
        _append("append_1", 1, 32, 8, 128),
        # the benchmark's prompt
        _append("append_2048", 2048, 32, 8, 128),
        # the float32 path: heads of another size, a number of tokens that is no multiple of anything
        _append("append_777_f32", 777, 16, 4, 96, "f32", 8),
        # a short prompt is read back
        _expand("expand_300", 1, 300, 8, 128),
        # a chunk's sequences, long contexts of unlike length
        _expand("expand_5x30000", 5, 30000, 8, 128),
        # one conversation: latency
        _attend("decode_1x900", 1, 900, 32, 8, 128),
        # the benchmark's decode batch
        _attend("decode_8x4096", 8, 4096, 32, 8, 128, least=1.0),
        # a busy server with long contexts of unlike length
        _attend("decode_64x8192", 64, 8192, 32, 8, 128),
        # the float32 path, heads of another size, small pages
        _attend("decode_33_f32", 33, 1111, 16, 2, 64, "f32", 8),
        # a window, eight query heads a kv head, heads of 64
        _attend("decode_21_window", 21, 5000, 64, 8, 64, window=1500),
        # a few tokens of each sequence, as short turns bring them
        _attend("turns_12x7", 12, 2600, 32, 8, 128, tokens=7),
        # a chunk of a long prompt
        _attend("chunk_512", 1, 6000, 32, 8, 128, tokens=512, least=1.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "expand", "attend", "attend"])
    f32 = rng.random() < 0.25
    dtype, page = "f32" if f32 else "bf16", rng.choice([4, 8, 16, 16, 32])
    dim = rng.choice([32, 64, 96, 128, 128, 256])
    heads, kv_heads = rng.choice([(32, 8), (16, 4), (8, 8), (40, 8), (32, 2), (24, 3)])
    if op == "append":
        return _unnamed(_append("", _log(rng, 1, 2048), heads, kv_heads, dim, dtype, page, rng.random() < 0.7, rng.choice([dim, dim, dim // 2, 0])))
    if op == "expand":
        seqs = _log(rng, 1, 40)
        return _unnamed(_expand("", seqs, _log(rng, 10, 100_000 // seqs), kv_heads, dim, dtype, page))
    tokens = rng.choice([1, 1, 1, 1, _log(rng, 2, 12), _log(rng, 13, 500)])
    seqs = _log(rng, 1, 60 if tokens == 1 else 16 if tokens <= 12 else 3)
    most = min(20_000, 150_000 // seqs) if tokens == 1 else min(8000, 60_000 // seqs, 12_000_000_000 // (tokens * seqs * heads * dim))
    keys = max(tokens, _log(rng, 40, max(41, most)))
    window = rng.choice([0, 0, 0, max(1, keys // 3)])
    return _unnamed(_attend("", seqs, keys, heads, kv_heads, dim, dtype, page, tokens, window, rng.choice([0.1, 0.5, 1.0])))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(shape, g, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=g)


def _on(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _host(g):
    return torch.Generator().manual_seed(int(torch.randint(0, 1 << 30, (1,), generator=g, device=DEVICE).item()))


def _pools(pages, case, g):
    """Codes and steps of groups whose values are about normal."""
    heads, page, dim = case["kv_heads"], case["page"], case["dim"]
    made = []
    for _ in range(2):
        codes = torch.randint(0, 256, (pages, heads, page, dim // 2), generator=g, device=DEVICE, dtype=torch.uint8)
        step = torch.empty((pages, heads, page, dim // GROUP, 1), device=DEVICE).uniform_(0.2, 0.36, generator=g)
        least = step * torch.empty_like(step).uniform_(-9.0, -6.0, generator=g)
        made += [codes, torch.cat([step, least], 4).flatten(3).to(torch.bfloat16)]
    return made


def _prepare_append(case, g):
    n, hq, hkv, dim, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype, rotary = TYPES[case["dtype"]], case["rotary"]
    host = _host(g)
    pages = -(-n // page)
    pools = _pools(pages + 3, case, g)
    table = torch.randperm(pages + 3, generator=host)[:pages]
    at = torch.arange(n)
    slots = table[at // page] * page + at % page
    angles = torch.arange(n, dtype=torch.float64).view(-1, 1) * 1e6 ** (-torch.arange(rotary // 2, dtype=torch.float64) / max(1, rotary // 2))
    weights = [(1 + 0.1 * _normal((dim,), g, torch.float32)) if case["norm"] else None for _ in range(2)]
    return dict(qkv=_normal((n, (hq + 2 * hkv) * dim), g, dtype, 2.0), q_out=torch.zeros((n, hq, dim), dtype=dtype, device=DEVICE), pools=pools, slots=slots.to(torch.int32).to(DEVICE),
                cos=angles.cos().float().to(DEVICE), sin=angles.sin().float().to(DEVICE), weights=weights, heads=hq, kv_heads=hkv, dim=dim, rotary=rotary, page=page,
                table=table.to(torch.int32).view(1, -1).to(DEVICE), kv_len=_on([n]), out=_expanded(case, pages), table_out=torch.full((1, pages), -1, dtype=torch.int32, device=DEVICE))


def _expanded(case, pages):
    """Pages that the values go to, nothing in them."""
    return [torch.zeros((pages, case["kv_heads"], case["page"], case["dim"]), dtype=TYPES[case["dtype"]], device=DEVICE) for _ in range(2)]


def _cache(case, g, lens):
    """Sequences of unlike length over pages in no order, and the pages of a window that have gone back to the pool."""
    page, host = case["page"], _host(g)
    counts = [-(-n // page) for n in lens]
    total = sum(counts)
    free = torch.randperm(total, generator=host).to(torch.int32)
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = free[at:at + n]
        at += n
    return _pools(total, case, g), table


def _lengths(case, g, least):
    host, n, most = _host(g), case["seqs"], case["keys"]
    low = max(1, int(least * most))
    return [most] + torch.randint(low, most + 1, (n - 1,), generator=host).tolist()


def _prepare_expand(case, g):
    lens = _lengths(case, g, 0.3)
    pools, table = _cache(case, g, lens)
    return dict(pools=pools, table=table.to(DEVICE), kv_len=_on(lens), out=_expanded(case, table.numel()), table_out=torch.full_like(table, -1).to(DEVICE), dim=case["dim"])


def _prepare_attend(case, g):
    tokens, page, window = case["tokens"], case["page"], case["window"]
    lens = [max(tokens, n) for n in _lengths(case, g, case["least"])]
    q_lens = [tokens] + [max(1, tokens - i % 3) for i in range(1, len(lens))] if tokens > 1 else [1] * len(lens)
    pools, table = _cache(case, g, lens)
    if window:
        for i, (n, q) in enumerate(zip(lens, q_lens)):
            table[i, :max(0, n - q - window + 1) // page] = -1
    rows, seq = sum(q_lens), torch.tensor([i for i, q in enumerate(q_lens) for _ in range(q)])
    cu = [0]
    for q in q_lens:
        cu.append(cu[-1] + q)
    place = torch.tensor([t for q in q_lens for t in range(q)])
    q = _normal((rows, case["heads"], case["dim"]), g, TYPES[case["dtype"]])
    return dict(q=q, out=torch.zeros_like(q), pools=pools, table=table.to(DEVICE), kv_len=_on(lens), cu_q=_on(cu), q_lens=q_lens, seq=seq.to(DEVICE), place=place.to(DEVICE), tokens=tokens,
                window=window or None, scale=case["dim"] ** -0.5)


def prepare(case, seed):
    g = _generator(seed)
    return dict({"append": _prepare_append, "expand": _prepare_expand, "attend": _prepare_attend}[case["op"]](case, g), op=case["op"])


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from pulsar_b200 import ops
    if s["op"] == "attend":
        one = s["tokens"] == 1
        ops.paged_attention_4bit(s["q"], *s["pools"], s["out"], s["table"], s["kv_len"], s["scale"], s["window"], None if one else s["cu_q"], None if one else s["q_lens"])
        return s["out"]
    if s["op"] == "append":
        ops.qk_norm_rope_write_4bit(s["qkv"], s["q_out"], *s["pools"], s["slots"], s["cos"], s["sin"], *s["weights"], EPS, s["heads"], s["kv_heads"], s["dim"], s["rotary"], s["page"])
        ops.expand_pages_4bit(*s["pools"], s["table"], s["kv_len"], *s["out"], s["table_out"])
        return [s["q_out"], *s["out"]]
    ops.expand_pages_4bit(*s["pools"], s["table"], s["kv_len"], *s["out"], s["table_out"])
    return [*s["out"], s["table_out"]]


# ------------------------------------------------------------------------------------------------ the plain form
def _next_bf16(b, up):
    """The next bfloat16 above (or below) each."""
    bits = b.view(torch.int16)
    away = (b > 0) | ((b == 0) & up) if up else (b < 0) | (b == 0)
    stepped = torch.where(away, (bits & 0x7fff) + 1, (bits & 0x7fff) - 1) | (bits & -0x8000)
    return stepped.to(torch.int16).view(torch.bfloat16)


def _quantised(x):
    """(codes, steps) of float64 values [..., D], in groups: [..., G, 32] and bfloat16 [..., G, 2]."""
    x = x.unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    least = low.to(torch.bfloat16)
    least = torch.where(least.double() > low, _next_bf16(least, False), least)
    wanted = (high - least.double()) / 15
    step = wanted.to(torch.bfloat16)
    step = torch.where(step.double() < wanted, _next_bf16(step, True), step)
    m, t = least.double().unsqueeze(-1), step.double().unsqueeze(-1)
    codes = torch.where(t > 0, torch.round((x - m) / torch.where(t > 0, t, 1.0)), 0.0).clamp(0, 15)
    return codes, torch.stack([step, least], -1)


def _packed(codes):
    """Bytes [..., D / 2] of codes [..., G, 32]."""
    c = codes.to(torch.uint8).unflatten(-1, (8, 4)).transpose(-3, -2)               # [..., 8, G, 4]
    return (c[..., 0::2] | c[..., 1::2] << 4).flatten(-3)


def _values(codes, steps):
    """float32 values [..., D] of bytes [..., D / 2] and steps [..., D / 16]."""
    groups = steps.shape[-1] // 2
    c = codes.unflatten(-1, (8, groups, 2))
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).transpose(-3, -2).flatten(-2)  # [..., G, 32]
    s = steps.float().unflatten(-1, (groups, 2))
    return (s[..., 1:] + s[..., :1] * c).flatten(-2)


def _turned(x, s, weight):
    """Normed and rotated heads [n, heads, dim], in 64 bits: a code is decided next to a border."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.double()
    half = s["rotary"] // 2
    c, t = s["cos"].double().unsqueeze(1), s["sin"].double().unsqueeze(1)
    u, v = x[..., :half], x[..., half:2 * half]
    return torch.cat([u * c - v * t, v * c + u * t, x[..., 2 * half:]], -1)


def _run_append(s):
    hq, hkv, dim, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    rows = s["qkv"].view(-1, hq + 2 * hkv, dim)
    s["q_out"].copy_(_turned(rows[:, :hq], s, s["weights"][0]))
    slots = s["slots"].long()
    k = _turned(rows[:, hq:hq + hkv], s, s["weights"][1]).to(rows.dtype)
    out = [s["q_out"]]
    for x, codes, steps, into in ((k, *s["pools"][:2], s["out"][0]), (rows[:, hq + hkv:], *s["pools"][2:], s["out"][1])):
        c, t = _quantised(x.double())
        codes[slots // page, :, slots % page] = _packed(c)
        steps[slots // page, :, slots % page] = t.flatten(-2)
        out.append(_expanded_into(codes, steps, s, into))
    return out


def _expanded_into(codes, steps, s, into):
    """Pages of the table's rows one behind the other; places that hold no key become zero, pages that hold none stay as they were."""
    table = s["table"].long()
    n, width = table.shape
    page = codes.shape[2]
    values = _values(codes[table.clamp_min(0)], steps[table.clamp_min(0)])                          # [n, width, heads, page, D]
    held = torch.arange(width * page, device=DEVICE).view(1, width, 1, page, 1) < s["kv_len"].view(-1, 1, 1, 1, 1)
    there = held[:, :, :, :1]
    return into.copy_(torch.where(there, torch.where(held, values, 0.0), into.view(values.shape).float()).flatten(0, 1))


def _run_expand(s):
    out = [_expanded_into(s["pools"][2 * i], s["pools"][2 * i + 1], s, s["out"][i]) for i in (0, 1)]
    table = s["table"]
    page = s["pools"][0].shape[2]
    place = torch.arange(table.numel(), dtype=torch.int32, device=DEVICE).view(table.shape)
    there = (torch.arange(table.shape[1], device=DEVICE) * page < s["kv_len"].view(-1, 1)) & (table >= 0)
    return [*out, s["table_out"].copy_(torch.where(there, place, -1))]


def _run_attend(s):
    table = s["table"].long().clamp_min(0)
    seqs, (rows, hq, dim), m = table.shape[0], s["q"].shape, s["tokens"]
    _, hkv, page, _ = s["pools"][0].shape
    keys = table.shape[1] * page
    k, v = (_values(s["pools"][i][table], s["pools"][i + 1][table]).transpose(1, 2).reshape(seqs, hkv, keys, dim) for i in (0, 2))
    q = torch.zeros((seqs, m, hq, dim), device=DEVICE)
    q[s["seq"], s["place"]] = s["q"].float()
    q = q.view(seqs, m, hkv, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, -1, dim)
    scores = (q @ k.transpose(2, 3) * s["scale"]).view(seqs, hkv, m, -1, keys)
    count = s["cu_q"][1:] - s["cu_q"][:-1]
    at = (s["kv_len"] - count).view(-1, 1) + torch.arange(m, device=DEVICE)                        # [seqs, m]: positions
    key = torch.arange(keys, device=DEVICE)
    seen = key <= at.unsqueeze(-1)
    if s["window"]:
        seen &= key > at.unsqueeze(-1) - s["window"]
    p = scores.masked_fill(~seen.view(seqs, 1, m, 1, keys), -math.inf)
    p = (p - p.amax(-1, keepdim=True).clamp_min(-3e38)).exp()
    o = (p.view(seqs, hkv, -1, keys) @ v).view(seqs, hkv, m, -1, dim) / p.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs, m, hq, dim)
    return s["out"].copy_(o[s["seq"], s["place"]])


def run(state):
    if own:
        return _run_own(state)
    return {"append": _run_append, "expand": _run_expand, "attend": _run_attend}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size, dim, hkv = TYPES[case["dtype"]].itemsize, case["dim"], case["kv_heads"]
    held = 2 * hkv * (dim // 2 + dim // 8)                                                          # a token's keys and values in 4 bits
    if case["op"] == "append":
        n, hq = case["tokens"], case["heads"]
        return {"bytes": n * ((2 * hq + 2 * hkv) * dim * size + 2 * held + 2 * hkv * dim * size + 4 * case["rotary"] + 4), "flops": 20 * n * (hq + 2 * hkv) * dim}
    if case["op"] == "expand":
        keys = case["keys"] * (1 + (case["seqs"] - 1) * 0.65)
        return {"bytes": keys * (held + 2 * hkv * dim * size), "flops": 4 * keys * hkv * dim}
    n, tokens, hq = case["seqs"], case["tokens"], case["heads"]
    mean = case["keys"] * (1 + (n - 1) * (1 + case["least"]) / 2)
    if case["window"]:
        mean = min(mean, n * (case["window"] + tokens))
    attended = tokens * max(n, mean - n * (tokens - 1) / 2)
    return {"bytes": mean * held + 2 * n * tokens * hq * dim * size, "flops": 4 * attended * hq * dim}


# ------------------------------------------------------------------------------------------------ 64 bits
def _read(codes, steps, dim):
    """float64 values [..., dim]: channel by channel from the words that hold them."""
    words = codes.contiguous().view(torch.int16).long() & 0xffff
    channel = torch.arange(dim, device=codes.device)
    g, i = channel // GROUP, channel % GROUP
    c = words.index_select(-1, (i // 4) * (dim // GROUP) + g) >> (4 * (i % 4)) & 15
    t = steps.double()
    return t.index_select(-1, 2 * g + 1) + t.index_select(-1, 2 * g) * c


def _near(x, dtype):
    """What a cache of 4 bits makes of ``x`` in ``dtype``, [..., dim] in 64 bits."""
    x = x.to(dtype).double().unflatten(-1, (-1, GROUP))
    low, high = x.aminmax(dim=-1, keepdim=True)

    def cut(v, up):            # to 8 bits, towards +inf or -inf
        mantissa, exponent = torch.frexp(v)
        whole = mantissa * 256
        return torch.ldexp(torch.ceil(whole) if up else torch.floor(whole), exponent - 8)
    m = cut(low, False)
    s = cut((high - m) / 15, True)
    return (m + s * torch.nan_to_num(torch.round((x - m) / s)).clamp(0, 15)).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    dim, page, hkv = case["dim"], case["page"], case["kv_heads"]
    if case["op"] == "append":
        n, hq, half, dtype = case["tokens"], case["heads"], case["rotary"] // 2, TYPES[case["dtype"]]
        rows = s["qkv"].double().view(n, hq + 2 * hkv, dim)
        parts = list(rows.split([hq, hkv, hkv], 1))
        for i, w in enumerate(s["weights"]):
            x = parts[i] if w is None else parts[i] * w.double() * (parts[i].pow(2).sum(-1, keepdim=True) / dim + EPS).rsqrt()
            pair = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.complex(s["cos"].double(), s["sin"].double()).unsqueeze(1)
            parts[i] = torch.cat([pair.real, pair.imag, x[..., 2 * half:]], -1)
        held = []
        for x in parts[1:]:
            full = torch.zeros((s["table"].shape[1] * page, hkv, dim), dtype=torch.float64, device=DEVICE)
            full[:n] = _near(x, dtype)
            held.append(full.view(-1, page, hkv, dim).transpose(1, 2).contiguous())
        return [parts[0], *held]
    if case["op"] == "expand":
        out = [torch.zeros(o.shape, dtype=torch.float64, device=DEVICE) for o in s["out"]]
        for i, n in enumerate(s["kv_len"].tolist()):
            count, first = -(-n // page), i * s["table"].shape[1]
            pages = s["table"][i, :count].long()
            for o, codes, steps in ((out[0], *s["pools"][:2]), (out[1], *s["pools"][2:])):
                o[first:first + count] = _read(codes[pages], steps[pages], dim)
                o[first + count - 1, :, n - (count - 1) * page:] = 0
        return [*out, None]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    at, group = 0, case["heads"] // hkv
    for i, (n, count) in enumerate(zip(s["kv_len"].tolist(), s["q_lens"])):
        first = max(0, n - count - case["window"] + 1) // page if case["window"] else 0
        pages = s["table"][i, first:-(-n // page)].long()
        k, v = (_read(s["pools"][j][pages], s["pools"][j + 1][pages], dim).transpose(0, 1).flatten(1, 2)[:, :n - first * page] for j in (0, 2))     # [kv heads, keys, dim]
        q = s["q"][at:at + count].double().view(count, hkv, group, dim)
        score = torch.einsum("thgd,hnd->thgn", q, k) * s["scale"]
        key, pos = torch.arange(first * page, n, device=DEVICE), torch.arange(n - count, n, device=DEVICE).view(-1, 1)
        seen = (key <= pos) & (key > pos - (case["window"] or n + 1))
        score = score.masked_fill(~seen.view(count, 1, 1, -1), -math.inf)
        out[at:at + count] = torch.einsum("thgn,hnd->thgd", torch.softmax(score, -1), v).reshape(count, case["heads"], dim)
        at += count
    return out
