"""Attention over a cache of 4 bits against bounds that shrink with the outputs (cache4_sharp): that those bounds notice a part that is lost, and that every
way to deal a call out stays within them."""
import types

import pytest
import torch
from cache4_sharp import beyond, expected
from test_attention_cache4 import DEALT, Case, dealt_out

from pulsar_b200 import ops

cuda = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]
FLOAT32 = [-1, -8, -4, -2, -2, -1, -2, 0, 0, 0, 0]            # how a call of float32 is dealt out: -n for a cluster of n blocks a head, 0 for even shares
DENSE = [([6000], [512], 32, 8, 128, 16, None), ([6000, 300], [130, 300], 8, 2, 128, 16, 1500), ([5000, 20, 900], [64, 20, 200], 16, 2, 64, 8, None)]


def of(lens, q_lens, hq, hkv, dim, page, window, dtype):
    return Case(lens, hq, hkv, dim, page, dtype, len(lens) + dim, q_lens, window=window)


def longest_alone(c):
    """The case's longest sequence by itself: (cache, its rows of q, its number of tokens)."""
    i = max((i for i, count in enumerate(c.q_lens) if count), key=lambda i: c.cache.lens[i])
    at = sum(c.q_lens[:i])
    cache = types.SimpleNamespace(tables=[c.cache.tables[i]], lens=[c.cache.lens[i]], pools=c.cache.pools, page=c.cache.page, hkv=c.cache.hkv)
    return cache, c.q[at:at + c.q_lens[i]], [c.q_lens[i]]


def left_out(c, keys, expanded=False):
    """(elements beyond the bound where nothing is wrong, where the outputs are zeros, where some keys in the middle of what is seen are left out, where they
    count twice), of the longest sequence."""
    cache, q, q_lens = longest_alone(c)
    n, count = cache.lens[0], q_lens[0]
    first = max(0, n - count - c.window + 1) if c.window else 0
    gone = max(first, (first + n - count) // 2 // keys * keys)
    without = {0: range(gone, min(n, gone + keys))}
    want, most = expected(cache, q, q_lens, c.scale, c.window, expanded=expanded)
    less, _ = expected(cache, q, q_lens, c.scale, c.window, without)
    # with their weights counted twice: w = sum of the left out's weights, out = (1 - w) less + w part, so that twice has out + w part over 1 + w
    part, _ = expected(cache, q, q_lens, c.scale, c.window, {0: [k for k in range(n) if k not in without[0]]})
    near = (part - less).square().sum(-1, keepdim=True).clamp_min(1e-30)
    w = ((want - less) * (part - less)).sum(-1, keepdim=True) / near
    twice = (want + w * part) / (1 + w)
    return [beyond(x.to(q.dtype), want, most) for x in (want, torch.zeros_like(want), less, twice)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens,q_lens,hq,hkv,dim,page,window,how", DEALT)
def test_a_lost_turn_of_keys_is_noticed(dtype, lens, q_lens, hq, hkv, dim, page, window, how):
    """32 keys: what a warp takes in a turn."""
    fine, zeros, less, twice = left_out(of(lens, q_lens, hq, hkv, dim, page, window, dtype), 32)
    assert fine == 0 and zeros > 0 and less > 0 and (twice > 0 or max(lens) <= 32)


@pytest.mark.parametrize("lens,q_lens,hq,hkv,dim,page,window", [DENSE[0][:2] + (8, 2) + DENSE[0][4:], *DENSE[1:]])
def test_a_lost_tile_of_expanded_keys_is_noticed(lens, q_lens, hq, hkv, dim, page, window):
    """128 keys, the tile of the dense kernels."""
    fine, zeros, less, twice = left_out(of(lens, [min(n, 64) for n in q_lens], hq, hkv, dim, page, window, torch.bfloat16), 128, True)
    assert fine == 0 and zeros > 0 and less > 0 and twice > 0


def check(c, expanded=False):
    got = c.run().cpu()
    want, most = expected(c.cache, c.q, c.q_lens, c.scale, c.window, expanded=expanded)
    assert torch.isfinite(got).all() and beyond(got, want, most) == 0, float(((got.double() - want).abs() / most.clamp_min(1e-30)).max())


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens,q_lens,hq,hkv,dim,page,window,how", DEALT)
def test_every_way_to_deal_a_call_out(monkeypatch, dtype, lens, q_lens, hq, hkv, dim, page, window, how):
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: False)
    c = of(lens, q_lens, hq, hkv, dim, page, window, dtype)
    if dtype == torch.float32:
        assert min(dealt_out(c, dtype), 0) == FLOAT32[DEALT.index((lens, q_lens, hq, hkv, dim, page, window, how))]
    check(c)


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hq,hkv,dim,page", [(32, 8, 128, 16), (8, 8, 64, 8), (12, 4, 96, 4), (2, 1, 256, 16), (6, 3, 32, 5), (3, 3, 160, 1), (8, 1, 192, 24), (36, 2, 224, 16)])
def test_sizes(monkeypatch, dtype, hq, hkv, dim, page):
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: False)
    for lens, q_lens, window in (([1, 17, 2000, 333], None, None), ([1, 17, 2000, 333], None, 100), ([500, 0, 64, 300], [20, 0, 1, 70], None), ([1600, 131], [70, 131], 500)):
        check(of(lens, q_lens, hq, hkv, dim, page, window, dtype))


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("scale", [6.0, -0.4, 0.0])
def test_scales(monkeypatch, dtype, scale):
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: False)
    for q_lens in (None, [9, 40, 1]):
        check(Case([200, 40, 3], 8, 2, 64, 16, dtype, 9, q_lens, scale=scale))


@cuda
@pytest.mark.parametrize("one", [True, False])
@pytest.mark.parametrize("lens,q_lens,hq,hkv,dim,page,window", DENSE)
def test_long_portions_either_way(monkeypatch, lens, q_lens, hq, hkv, dim, page, window, one):
    for expanded in (True, False):
        monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: expanded)
        monkeypatch.setattr(ops, "_one_head_a_block", lambda *a: one and dim == 128)
        check(of(lens, q_lens, hq, hkv, dim, page, window, torch.bfloat16), expanded)
