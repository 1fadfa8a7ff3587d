"""The operators of several scored continuations of one prompt, as their users call them.

  copy      ``ops.copy_pages``: pages of a cache's pools copied within the pools (a fork's last page) or into other pools (a cache
            that is made larger or smaller)
  scores    ``ops.token_scores``: log probability and rank of given tokens, entropy and the likeliest alternatives, from logits
  head      ``ops.head_scores``: log probability of given tokens and entropy straight from hidden rows and the head's weight
  shared    ``ops.paged_attention_shared``: attention of one token per sequence over a forked cache, where the pages that a family of
            sequences shares are read once

Where ``own`` is false, ``run`` computes the same from elementary operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda"
PAGE = 16
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _copy(name, entries, heads, widths, pages, copied, within, dtype="bf16", page=PAGE):
    return dict(name=name, op="copy", entries=entries, heads=heads, widths=widths, pages=pages, copied=copied, within=within, dtype=dtype, page=page)


def _scores(name, rows, vocab, top, dtype="f32", masked=0.0):
    return dict(name=name, op="scores", rows=rows, vocab=vocab, top=top, dtype=dtype, masked=masked)


def _head(name, rows, width, vocab, dtype="bf16", scale=1.0, cap=0.0):
    return dict(name=name, op="head", rows=rows, width=width, vocab=vocab, dtype=dtype, scale=scale, cap=cap)


def _shared(name, families, members, shared, own_keys, heads, kv_heads, dim, dtype="bf16", page=PAGE, alone=0):
    return dict(name=name, op="shared", families=families, members=members, shared=shared, own_keys=own_keys, heads=heads, kv_heads=kv_heads,
                dim=dim, dtype=dtype, page=page, alone=alone)


def listed():
    return [
        # a prompt of the benchmark's model is forked once: one page of every layer's keys and values
        _copy("fork_one", 36, 8, "128,128", 64, 1, True),
        # 32 continuations of one prompt begin
        _copy("fork_32", 36, 8, "128,128", 128, 32, True),
        # the benchmark's cache, 16,000 tokens held, moves into a pool of another size
        _copy("resize_1000", 36, 8, "128,128", 1100, 1000, False),
        # a token of one conversation, with its alternatives: latency
        _scores("scores_1", 1, 151936, 5),
        # a busy server's step
        _scores("scores_64", 64, 151936, 20),
        # a chunk of a prompt that is scored with alternatives; an odd vocabulary, most of it forbidden by a grammar in some rows
        _scores("scores_777_odd", 777, 32003, 8, "bf16", 0.3),
        # a line of text is scored without alternatives: bound by the head's weight
        _head("head_17", 17, 4096, 151936),
        # the benchmark's prompt is scored
        _head("head_2048", 2048, 4096, 151936),
        # the float32 path, a head with a scale and a cap
        _head("head_96_f32", 96, 1024, 32003, "f32", 0.5, 30.0),
        # eight continuations of one long prompt at the benchmark's sizes
        _shared("shared_8", 1, 8, 3840, 200, 32, 8, 128),
        # a busy server: 12 prompts with 8 continuations each, of unlike length, and 5 requests that share nothing
        _shared("shared_101_ragged", 12, 8, 2600, 500, 32, 8, 128, alone=5),
        # the float32 path, heads of another size
        _shared("shared_6_f32", 2, 3, 700, 90, 16, 4, 96, "f32", 8),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _vocabulary(rng, high):
    """Any number, most of them no multiple of a block (the listed cases have one that is)."""
    n = _log(rng, 257, high)
    return n + 1 if n % 512 == 0 else n


def draw(rng):
    op = rng.choice(["copy", "scores", "head", "shared"])
    if op == "copy":
        copied = _log(rng, 1, 900)
        within = rng.random() < 0.5
        widths = rng.choice(["128,128", "64,64", "576", "96,40", "512,64"])
        return _unnamed(_copy("", rng.randint(1, 36), rng.choice([1, 2, 4, 8]), widths, (2 * copied if within else copied) + rng.randint(1, 60), copied, within,
                              rng.choice(["bf16", "bf16", "f32"]), rng.choice([4, 8, 16])))
    if op == "scores":
        rows = _log(rng, 1, 900)
        return _unnamed(_scores("", rows, _vocabulary(rng, min(152000, 55_000_000 // rows)), rng.choice([0, 1, 5, 8, 20]), rng.choice(["f32", "f32", "bf16"]), rng.choice([0.0, 0.0, 0.5])))
    if op == "head":
        f32 = rng.random() < 0.25
        rows = _log(rng, 1, 200 if f32 else 2048)
        width = 8 * _log(rng, 8, 128 if f32 else 380)
        scale, cap = rng.choice([(1.0, 0.0), (1.0, 0.0), (0.5, 30.0)])
        return _unnamed(_head("", rows, width, _vocabulary(rng, 32003 if f32 else 152000), "f32" if f32 else "bf16", scale, cap))
    f32 = rng.random() < 0.25
    families, members = _log(rng, 1, 3 if f32 else 12), _log(rng, 2, 4 if f32 else 20)
    page = rng.choice([8, 16])
    most = min(3000, 40_000 // (families * members)) if not f32 else 900
    heads, kv_heads = rng.choice([(32, 8), (16, 4), (8, 8), (40, 8)])
    return _unnamed(_shared("", families, members, page * _log(rng, 1, max(2, most // page)), _log(rng, 1, 500), heads, kv_heads,
                            rng.choice([32, 96, 128] if f32 else [64, 128]), "f32" if f32 else "bf16", page, rng.choice([0, 0, 1, 5])))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _widths(case):
    return [int(w) for w in case["widths"].split(",")]


def _pool_shape(case, width, pages):
    return case["entries"], pages, case["heads"], case["page"], width


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(shape, g, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=g)


def _prepare_copy(case, g):
    pools = [_normal(_pool_shape(case, w, case["pages"]), g, TYPES[case["dtype"]]) for w in _widths(case)]
    order = torch.randperm(case["pages"], generator=g, device=DEVICE).to(torch.int32)
    n = case["copied"]
    src = order[:n].contiguous()
    if case["within"]:                       # no page is both read and written
        into, dst = pools, order[n:2 * n].contiguous()
    else:
        into = [torch.zeros(_pool_shape(case, w, n + 7), dtype=TYPES[case["dtype"]], device=DEVICE) for w in _widths(case)]
        dst = torch.arange(n, dtype=torch.int32, device=DEVICE)
    return dict(pools=pools, into=into, src=src, dst=dst)


def _prepare_scores(case, g):
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    logits = _normal((rows, vocab), g, TYPES[case["dtype"]], 2.5)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
    if case["masked"]:                       # rows in which nine tokens of ten are forbidden, not the given one
        forbidden = torch.rand((rows, 1), generator=g, device=DEVICE) < case["masked"]
        keep = torch.rand((rows, vocab), generator=g, device=DEVICE) < 0.1
        keep.scatter_(1, tokens.view(-1, 1), True)
        logits.masked_fill_(forbidden & ~keep, -math.inf)
    made = dict(logits=logits, tokens=tokens.to(torch.int32), logprob=torch.empty(rows, device=DEVICE), entropy=torch.empty(rows, device=DEVICE),
                rank=torch.empty(rows, dtype=torch.int32, device=DEVICE), top_ids=None, top_logprob=None)
    if top:
        made.update(top_ids=torch.empty((rows, top), dtype=torch.int32, device=DEVICE), top_logprob=torch.empty((rows, top), device=DEVICE))
    return made


def _prepare_head(case, g):
    rows, width, vocab = case["rows"], case["width"], case["vocab"]
    dtype = TYPES[case["dtype"]]
    h = _normal((rows, width), g, dtype)                                     # as a norm leaves them
    w = _normal((vocab, width), g, dtype, 0.02)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE).to(torch.int32)
    return dict(h=h, w=w, tokens=tokens, logprob=torch.empty(rows, device=DEVICE), entropy=torch.empty(rows, device=DEVICE),
                scale=case["scale"], cap=case["cap"] or None)


def _prepare_shared(case, g):
    page, hkv, dim = case["page"], case["kv_heads"], case["dim"]
    dtype = TYPES[case["dtype"]]
    host = torch.Generator().manual_seed(int(torch.randint(0, 1 << 30, (1,), generator=g, device=DEVICE).item()))
    sizes = [case["members"]] * case["families"] + [1] * case["alone"]
    shared_pages, own_lens = [], []
    most = case["shared"] // page
    for f, size in enumerate(sizes):         # unlike prompts: half of the longest to all of it; a lone request shares nothing
        shared_pages.append(0 if size == 1 else most if f == 0 else int(torch.randint(max(1, most // 2), most + 1, (1,), generator=host)))
        longest = case["own_keys"] if size > 1 else case["own_keys"] + case["shared"] // 2
        own_lens.append([longest if f == 0 and m == 0 else int(torch.randint(1, longest + 1, (1,), generator=host)) for m in range(size)])
    total = sum(shared_pages) + sum(-(-n // page) for lens in own_lens for n in lens)
    free = torch.randperm(total, generator=host).tolist()
    tables, kv_len, shared_len, members, starts = [], [], [], [], [0]
    for n_shared, lens in zip(shared_pages, own_lens):
        prefix = [free.pop() for _ in range(n_shared)]
        for n in lens:
            tables.append(prefix + [free.pop() for _ in range(-(-n // page))])
            kv_len.append(n_shared * page + n)
            shared_len.append(n_shared * page)
        if n_shared:
            members += range(len(kv_len) - len(lens), len(kv_len))
            starts.append(len(members))
    width = max(len(t) for t in tables)
    on = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)                               # noqa: E731
    k, v = (_normal((total, hkv, page, dim), g, dtype) for _ in range(2))
    q = _normal((len(tables), case["heads"], dim), g, dtype)
    return dict(q=q, k=k, v=v, out=torch.empty_like(q), table=on([t + [-1] * (width - len(t)) for t in tables]), kv_len=on(kv_len), shared_len=on(shared_len),
                members=on(members), starts=on(starts), most_members=case["members"], most_shared=max(shared_len), scale=dim ** -0.5)


def prepare(case, seed):
    g = _generator(seed)
    made = {"copy": _prepare_copy, "scores": _prepare_scores, "head": _prepare_head, "shared": _prepare_shared}[case["op"]](case, g)
    return dict(made, op=case["op"])


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from pulsar_b200 import ops
    if s["op"] == "copy":
        ops.copy_pages(s["pools"], s["into"], s["src"], s["dst"])
        return s["into"]
    if s["op"] == "scores":
        ops.token_scores(s["logits"], s["tokens"], s["logprob"], s["entropy"], s["rank"], s["top_ids"], s["top_logprob"])
        return [s["logprob"], s["entropy"], s["rank"], s["top_ids"], s["top_logprob"]]
    if s["op"] == "head":
        ops.head_scores(s["h"], s["w"], s["tokens"], s["logprob"], s["entropy"], s["scale"], s["cap"])
        return [s["logprob"], s["entropy"]]
    ops.paged_attention_shared(s["q"], s["k"], s["v"], s["out"], s["table"], s["kv_len"], s["shared_len"], s["members"], s["starts"],
                               s["most_members"], s["most_shared"], s["scale"])
    return s["out"]


# ------------------------------------------------------------------------------------------------ the plain form
def _log_softmax_sums(x):
    """(x - lse, entropy) of float32 rows; a forbidden token, of logit -inf, adds nothing."""
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    total = e.sum(1, keepdim=True)
    entropy = total.log() - (e * d.clamp_min(-3e38)).sum(1, keepdim=True) / total
    return d - total.log(), entropy.squeeze(1)


def _run_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    return [into.index_copy_(1, dst, pool.index_select(1, src)) for pool, into in zip(s["pools"], s["into"])]


def _run_scores(s):
    x, tokens = s["logits"].float(), s["tokens"].long().view(-1, 1)
    log_p, entropy = _log_softmax_sums(x)
    given = x.gather(1, tokens)
    place = torch.arange(x.shape[1], device=x.device)
    rank = ((x > given) | ((x == given) & (place < tokens))).sum(1).to(torch.int32)
    if s["top_ids"] is None:
        return [log_p.gather(1, tokens).squeeze(1), entropy, rank, None, None]
    bits = (x + 0.0).view(torch.int32).long()                # larger number, larger key; of equal ones the lower place
    key = torch.where(bits >= 0, bits, -(bits & 0x7fffffff)) * (1 << 31) - place
    ids = key.topk(s["top_ids"].shape[1], dim=1).indices
    return [log_p.gather(1, tokens).squeeze(1), entropy, rank, ids.to(torch.int32), log_p.gather(1, ids)]


def _run_head(s):
    x = s["h"].float() @ s["w"].float().t() * s["scale"]
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    log_p, entropy = _log_softmax_sums(x)
    return [log_p.gather(1, s["tokens"].long().view(-1, 1)).squeeze(1), entropy]


def _run_shared(s):
    q, table = s["q"], s["table"].long().clamp_min(0)
    n, heads, dim = q.shape
    _, hkv, page, _ = s["k"].shape
    keys = table.shape[1] * page
    k, v = (pool[table].float().transpose(1, 2).reshape(n, hkv, keys, dim) for pool in (s["k"], s["v"]))
    scores = q.float().view(n, hkv, heads // hkv, dim) @ k.transpose(2, 3) * s["scale"]
    beyond = torch.arange(keys, device=q.device) >= s["kv_len"].view(-1, 1)
    p = (scores.masked_fill(beyond.view(n, 1, 1, keys), -math.inf))
    p = (p - p.amax(3, keepdim=True)).exp()
    return ((p @ v) / p.sum(3, keepdim=True)).reshape(n, heads, dim).to(q.dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"copy": _run_copy, "scores": _run_scores, "head": _run_head, "shared": _run_shared}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "copy":
        moved = sum(_widths(case)) * case["entries"] * case["heads"] * case["page"] * size * case["copied"]
        return {"bytes": 2 * moved + 8 * case["copied"], "flops": 0}
    if case["op"] == "scores":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * vocab * size + rows * (16 + 8 * case["top"]), "flops": 6 * rows * vocab}
    if case["op"] == "head":
        rows, width, vocab = case["rows"], case["width"], case["vocab"]
        return {"bytes": (rows + vocab) * width * size + 12 * rows, "flops": 2 * rows * vocab * width + 6 * rows * vocab}
    # prompts are half of the longest to all of it, own keys one to the most (means)
    families, members, alone = case["families"], case["members"], case["alone"]
    shared = case["shared"] + (families - 1) * 0.75 * case["shared"]
    lone = alone * 0.5 * (case["own_keys"] + case["shared"] // 2)
    separate = families * members * 0.5 * case["own_keys"] + lone
    n = families * members + alone
    row = 2 * case["kv_heads"] * case["dim"] * size
    attended = members * shared + separate
    return {"bytes": (shared + separate) * row + 2 * n * case["heads"] * case["dim"] * size, "flops": 4 * attended * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_rows(x, tokens, top):
    """Rows of float64 logits: log probability of the token, entropy, and the log probabilities of the likeliest."""
    lse = torch.logsumexp(x, 1)
    p = torch.softmax(x, 1)
    entropy = -torch.special.xlogy(p, p).sum(1)
    best = torch.topk(x, top, dim=1).values - lse.view(-1, 1) if top else None
    return x[torch.arange(x.shape[0], device=x.device), tokens.long()] - lse, entropy, best


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        for pool, into in zip(s["pools"], s["into"]):
            before = pool.clone() if case["within"] else pool
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                into[:, b] = before[:, a]
        return s["into"]
    if case["op"] == "scores":
        parts = [_exact_rows(s["logits"][i:i + 64].double(), s["tokens"][i:i + 64], case["top"]) for i in range(0, case["rows"], 64)]
        logprob, entropy = (torch.cat([p[k] for p in parts]) for k in (0, 1))
        return [logprob, entropy, None, None, torch.cat([p[2] for p in parts]) if case["top"] else None]
    if case["op"] == "head":
        w = s["w"].double()
        parts = []
        for i in range(0, case["rows"], 256):
            x = case["scale"] * torch.mm(s["h"][i:i + 256].double(), w.t())
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            parts.append(_exact_rows(x, s["tokens"][i:i + 256], 0))
        return [torch.cat([p[k] for p in parts]) for k in (0, 1)]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    group = case["heads"] // case["kv_heads"]
    for i, n in enumerate(s["kv_len"].tolist()):
        pages = s["table"][i, :-(-n // case["page"])].long()
        k, v = (torch.cat(list(pool[pages].double()), dim=1)[:, :n] for pool in (s["k"], s["v"]))      # [kv heads, n, dim]
        q = s["q"][i].double().view(case["kv_heads"], group, case["dim"])
        out[i] = torch.einsum("hgn,hnd->hgd", torch.softmax(s["scale"] * torch.einsum("hgd,hnd->hgn", q, k), -1), v).reshape(case["heads"], case["dim"])
    return out
