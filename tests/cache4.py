"""What the tests of the cache of 4 bits share: the format in 64 bits, written from its definition."""
import math
import random

import torch

GROUP = 32


def on(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cut_to_8_bits(v, up):
    """float64 values to 8 significant bits, towards +inf or -inf; what lies below bfloat16's normal range has its fixed step."""
    mantissa, exponent = torch.frexp(v)
    exponent = exponent.clamp_min(-125).double()            # 2^-126 is the smallest normal number, 2^-133 the step below it
    whole = torch.ldexp(v, 8 - exponent)
    return torch.ldexp(torch.ceil(whole) if up else torch.floor(whole), exponent - 8)


def quantised(x):
    """(codes [..., G, 32], step [..., G], least [..., G]) of float64 values [..., D]."""
    x = x.unflatten(-1, (-1, GROUP))
    least = cut_to_8_bits(x.amin(-1), False)
    step = cut_to_8_bits((x.amax(-1) - least) / 15, True)
    quotient = (x - least.unsqueeze(-1)) / torch.where(step > 0, step, 1.0).unsqueeze(-1)
    return torch.round(quotient).clamp(0, 15), step, least


def words_of(codes):
    """Bytes [..., D / 2]: word r * G + g holds channels 32 g + 4 r .. + 3, the first in the lowest bits."""
    groups = codes.shape[-2]
    words = torch.zeros((*codes.shape[:-2], 8 * groups), dtype=torch.int64)
    for g in range(groups):
        for i in range(GROUP):
            words[..., i // 4 * groups + g] |= codes[..., g, i].long() << (4 * (i % 4))
    return torch.stack([words & 255, words >> 8], -1).flatten(-2).to(torch.uint8)


def steps_of(step, least):
    return torch.stack([step, least], -1).flatten(-2).to(torch.bfloat16)


def values_of(codes, steps):
    """float64 values [..., D] of bytes and steps."""
    groups = steps.shape[-1] // 2
    out = torch.zeros((*codes.shape[:-1], GROUP * groups), dtype=torch.float64)
    for g in range(groups):
        for i in range(GROUP):
            c = codes[..., 2 * (i // 4 * groups + g) + i % 4 // 2].long() >> (4 * (i % 2)) & 15
            out[..., GROUP * g + i] = steps[..., 2 * g + 1].double() + steps[..., 2 * g].double() * c
    return out


class Cache4:
    """Sequences of lengths ``lens`` over pages in no order.  Steps of places that no key holds are ``beyond``; ids of pages behind a window
    are -1, or ``stray`` where given."""

    def __init__(self, lens, hkv, dim, page, seed, beyond=float("nan"), spare=3):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.lens, self.page, self.dim, self.hkv = list(lens), page, dim, hkv
        counts = [-(-n // page) for n in lens]
        total = sum(counts) + spare
        free = list(range(total))
        rng.shuffle(free)
        self.tables = [[free.pop() for _ in range(n)] for n in counts]
        self.pools = []
        for _ in range(2):
            codes = torch.randint(0, 256, (total, hkv, page, dim // 2), generator=g, dtype=torch.uint8)
            step = 0.2 + 0.16 * torch.rand((total, hkv, page, dim // GROUP), generator=g)
            least = -step * (6 + 3 * torch.rand(step.shape, generator=g))
            steps = steps_of(step, least)
            held = torch.zeros((total, page), dtype=torch.bool)
            for table, n in zip(self.tables, lens):
                for i, p in enumerate(table):
                    held[p, :n - i * page] = True
            steps.masked_fill_(~held.view(total, 1, page, 1), beyond)
            self.pools += [codes, steps]

    def table(self, width=0, stray=-1):
        width = max([1, width] + [len(t) for t in self.tables])
        return torch.tensor([t + [stray] * (width - len(t)) for t in self.tables], dtype=torch.int32)

    def key_values(self, i):
        """float64 keys and values [Hkv, n, D] of sequence i."""
        pages = self.tables[i]
        got = []
        for j in (0, 2):
            v = values_of(self.pools[j][pages], self.pools[j + 1][pages])                                # [pages, Hkv, page, D]
            got.append(v.transpose(0, 1).flatten(1, 2)[:, :self.lens[i]])
        return got


def attended(cache, q, q_lens, scale, window=None):
    """(softmax(scale q k) v in 64 bits, a bound on the scores' size, on the values') for the rows of sequences one behind the other."""
    n, hq, dim = q.shape
    out = torch.zeros(n, hq, dim, dtype=torch.float64)
    at, score_size, value_size = 0, 0.0, 0.0
    for i, count in enumerate(q_lens):
        length = cache.lens[i]
        if length and count:
            k, v = (x.repeat_interleave(hq // cache.hkv, 0) for x in cache.key_values(i))
            rows = q[at:at + count].double()
            score = scale * torch.einsum("thd,hnd->thn", rows, k)
            pos, key = torch.arange(length - count, length).view(-1, 1, 1), torch.arange(length)
            seen = (key <= pos) & ((key > pos - window) if window else (key >= 0))
            p = torch.softmax(score.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
            out[at:at + count] = torch.einsum("thn,hnd->thd", p, v)
            least, step = (cache.pools[1][cache.tables[i]][..., j::2].double().nan_to_num(0.0).abs().max() for j in (1, 0))
            score_size = max(score_size, abs(scale) * float(rows.abs().sum(-1).max() * (least + 16 * step)))
            value_size = max(value_size, float(v.abs().max()))
        at += count
    return out, score_size, value_size


def bound(want, score_size, value_size, dtype, longest):
    """How far a result may be off.  A score is a sum of at most 256 products of a query's element with a step and a code, of no more than
    score_size together; the kernels multiply codes that stand at 1,024 and more (an offset which is taken off again), so that up to 1,040 / 16
    = 65 times score_size goes through float32 sums of 32 products each and a handful of sums of those.  The exponentials of the weights carry
    that over to the values' size, above and below the line; a sum of weights has up to longest / 8 terms a lane.  float32: codes stand about
    zero, no offset.  bfloat16: weights are rounded to 8 bits before their product with steps and codes, the result is."""
    unit = 2.0 ** -24
    through = score_size * (80 * 65 if dtype == torch.bfloat16 else 300)
    off = value_size * unit * (2 * through + longest / 8 + 64)
    if dtype == torch.bfloat16:
        return off + 2 * value_size * 2.0 ** -8 + want.abs() * 2.0 ** -8
    return off + want.abs() * unit
