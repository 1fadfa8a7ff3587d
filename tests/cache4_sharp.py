"""Attention over a cache of 4 bits in 64 bits, with how far every element of a kernel's output may be off.

out_c = sum_j p_j v_jc with sum_j p_j = 1.  A rounding moves one term of such a sum; the roundings of different keys and channels are independent
of one another and up or down alike, so that a sum of them stays below MANY times the root of the sum of their squares (Hoeffding: with 6.5 times
exceeded once in 7e8 elements).  That bound shrinks with the number of keys as the outputs themselves do, by the root, where the sum of the roundings' sizes
would not.  What is rounded, each by half a step (bfloat16 2^-8, float32 2^-24; sums inside the products cut off, a whole step 2^-23 of the
largest term):

  codes     the weight times the step, an operand of the second product, with c - 8 for its code: p_j s_j (c_j - 8)   (bfloat16 in one term;
            float32 in three, 2^-24 left over, and 2^-22 of the exponential)
            a score, which moves its weight and so out by p_j (v_jc - out_c): two products a group of 17 terms each, lined up in bfloat16 by codes
            that stand at 2^-14 where the bits of one are 2^-24 (2^11 for a code of one), in float32 three times as many by codes of up to 8; and
            3 G + 8 roundings of the whole score, which is no more than scale sum |q| (|m| + 16 s)
            the second product's sums: in bfloat16 136 times a fold of 128 keys' weights, of 16 products; in float32 8 times the weights, of all
  expanded  keys and values as bfloat16, the weights too
  either    the output; float32 sums of the weights and least values
"""
import math

import torch

from cache4 import GROUP, values_of

MANY = 6.5


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _of_sequence(cache, i):
    """float64 keys, values [Hkv, n, D], values' middles m + 8 s and steps [Hkv, n, D], and the largest step and least value of the keys."""
    pages, n, got = cache.tables[i], cache.lens[i], []
    for j in (0, 2):
        steps = cache.pools[j + 1][pages].double()
        step, least = (steps[..., e::2].repeat_interleave(GROUP, -1) for e in (0, 1))
        got.append([x.transpose(0, 1).flatten(1, 2)[:, :n] for x in (values_of(cache.pools[j][pages], cache.pools[j + 1][pages]), least + 8 * step, step, least)])
    (k, _, k_step, k_least), (v, middle, v_step, _) = got
    return k, v, middle, v_step, k_step, k_least


def expected(cache, q, q_lens, scale, window=None, hidden=None, expanded=False):
    """(outputs in 64 bits, how far each may be off), both [N, Hq, D].  ``hidden``: of sequence i, the keys that nobody sees."""
    rows, hq, dim = q.shape
    hkv, dtype = cache.hkv, q.dtype
    want, most = torch.zeros(rows, hq, dim, dtype=torch.float64), torch.zeros(rows, hq, dim, dtype=torch.float64)
    single, unit, cut, groups = dtype == torch.bfloat16, half_step(torch.float32), 2.0 ** -23, dim // GROUP
    at = 0
    for i, count in enumerate(q_lens):
        n = cache.lens[i]
        if n and count:
            k, v, middle, v_step, k_step, k_least = _of_sequence(cache, i)
            pos, key = torch.arange(n - count, n).view(-1, 1), torch.arange(n)
            seen = (key <= pos) & ((key > pos - window) if window else (key >= 0))
            if hidden is not None and i in hidden:
                seen = seen & ~torch.isin(key, torch.tensor(list(hidden[i])))
            seen = seen.view(1, count, 1, n)
            x = q[at:at + count].double().view(count, hkv, hq // hkv, dim).transpose(0, 1)                              # [Hkv, t, group, D]
            score = scale * torch.einsum("htgd,hnd->htgn", x, k)
            p = torch.softmax(score.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
            out = torch.einsum("htgn,hnd->htgd", p, v)
            squares = p.square()

            def rss(weights, of):
                """The root of sum_j (weights_j of_jc)^2."""
                return torch.einsum("htgn,hnd->htgd", weights, of.square()).clamp_min(0).sqrt()
            any_seen = seen.any(2).any(1)[0] if count else None
            step, least = float((k_step * any_seen.view(1, n, 1)).abs().max()), float((k_least * any_seen.view(1, n, 1)).abs().max())
            size = abs(scale) * x.abs().sum(-1) * (least + 16 * step)                                                # of a score's terms together
            largest = abs(scale) * x.abs().amax(-1) * step                                                           # of a product with a code of one
            # sum_j p_j^2 (v_jc - out_c)^2
            spread = (torch.einsum("htgn,hnd->htgd", squares, v.square()) - 2 * out * torch.einsum("htgn,hnd->htgd", squares, v) + out.square() * squares.sum(-1, keepdim=True))
            spread = spread.clamp_min(0).sqrt() + 1e-12 * out.abs()
            held, weight = torch.einsum("htgn,hnd->htgd", p, v.abs()), squares.sum(-1, keepdim=True).sqrt()
            scores = (3 * groups + 8) * unit * size + 4 * unit
            if expanded:
                rounded = 0.0
                for h in range(hkv):                                                # (q_i k_i)^2 summed over channels: the largest of any key
                    rounded = max(rounded, float(torch.einsum("tgd,nd->tgn", x[h].square(), k[h].square()).masked_fill(~seen[0], 0.0).amax().sqrt()))
                scores = scores + abs(scale) * half_step(torch.bfloat16) * rounded + math.sqrt(17 * dim / 16) * cut * size
                off = scores.unsqueeze(-1) * spread + 2 * half_step(torch.bfloat16) * rss(squares, v) + cut * math.sqrt(17 * (n / 16 + 1)) * held
            else:
                scores = scores + math.sqrt(34 * groups * (1 if single else 3)) * cut * largest * (2 ** 11 if single else 8)
                off = scores.unsqueeze(-1) * spread + (half_step(torch.bfloat16) if single else 4 * unit) * rss(squares, v - middle)
                of_value = float(v_step.nan_to_num(0.0).abs().max())
                off = off + (math.sqrt(272) * cut * 136 * of_value * math.sqrt(128) * weight if single else math.sqrt(51 * (n / 16 + 1)) * cut * 8 * of_value)
            off = MANY * (off + unit * (math.sqrt(n) + 32) * held) + half_step(dtype) * out.abs()
            want[at:at + count] = out.transpose(0, 1).reshape(count, hq, dim)
            most[at:at + count] = off.transpose(0, 1).reshape(count, hq, dim)
        at += count
    return want, most


def pages_hidden(cache, holes):
    """``hidden`` of ``expected`` for pages {sequence: logical pages} that are none."""
    return {i: [key for p in pages for key in range(p * cache.page, min((p + 1) * cache.page, cache.lens[i]))] for i, pages in holes.items()}


def beyond(got, want, most):
    """Elements that are further off than they may be (NaN among them)."""
    return int((~((got.double() - want).abs() <= most)).sum())
