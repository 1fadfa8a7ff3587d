"""Keys and values of a cache of 4 bits that are no numbers, in portions of many sequences over expanded pages and on codes: they reach the queries that see
them, and no others, of their own sequence or of one whose tiles are worked on later."""
import pytest
import torch
from cache4_sharp import beyond, expected
from test_attention_cache4 import Case

from pulsar_b200 import ops

cuda = pytest.mark.gpu
SIZES = [(32, 4, 128, 16), (3, 3, 128, 8), (32, 4, 64, 16), (16, 2, 128, 64)]
# many more tiles of tokens and heads than there are SMs, so that a block's buffers hold what it had of another sequence; sequences that end inside a tile of 128 keys
LENS = [300, 40] + [150 + 3 * i for i in range(40)]
TOKENS = [200, 30] + [20 + i for i in range(40)]


def case(hq, hkv, dim, page, window=None):
    return Case(LENS, hq, hkv, dim, page, torch.bfloat16, dim + page, TOKENS, window=window)


def sees(c, seq, key):
    """Rows of the batch that see ``key`` of sequence ``seq``."""
    rows = torch.zeros(len(c.q), dtype=torch.bool)
    at = sum(c.q_lens[:seq])
    for t in range(c.q_lens[seq]):
        pos = c.cache.lens[seq] - c.q_lens[seq] + t
        rows[at + t] = key <= pos and (not c.window or key > pos - c.window)
    return rows


def spoil(c, pool, seq, key, head, group, value):
    page, place = c.cache.tables[seq][key // c.cache.page], key % c.cache.page
    c.cache.pools[pool][page, head, place, 2 * group + 1] = value
    return sees(c, seq, key)


@cuda
@pytest.mark.parametrize("expanded", [True, False])
@pytest.mark.parametrize("window", [None, 70])
@pytest.mark.parametrize("pool", [1, 3])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("hq,hkv,dim,page", SIZES)
def test_no_number_reaches_a_query_that_does_not_see_it(monkeypatch, hq, hkv, dim, page, pool, value, window, expanded):
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: expanded)
    for one in (True, False) if expanded and dim == 128 else (False,):
        monkeypatch.setattr(ops, "_one_head_a_block", lambda *a: one)
        want, c = case(hq, hkv, dim, page, window).run().cpu(), case(hq, hkv, dim, page, window)
        rows = torch.zeros(len(c.q), dtype=torch.bool)
        for seq, key in ((0, 290), (0, 170), (1, 33), (20, 180)):                            # places behind the last are still NaN in the pool
            rows |= spoil(c, pool, seq, key, 1, 1, value)
        got = c.run().cpu()
        hit = torch.zeros(len(c.q), hq, dtype=torch.bool)
        hit[:, hq // hkv:2 * hq // hkv] = rows.view(-1, 1)
        if expanded:
            assert torch.equal(got[~hit], want[~hit])
        else:                                   # rows of a block move their maxima together: the others may be rounded elsewhere
            good = case(hq, hkv, dim, page, window)
            exact, most = expected(good.cache, good.q, good.q_lens, good.scale, window)
            assert beyond(got[~hit], exact[~hit], most[~hit]) == 0
        if value != value:
            of = got[hit][:, 32:64] if pool == 3 else got[hit]
            assert rows.any() and torch.isnan(of).all()


@cuda
@pytest.mark.parametrize("hq,hkv,dim,page", SIZES)
def test_values_past_the_end_of_bfloat16_reach_no_other_query(monkeypatch, hq, hkv, dim, page):
    """A least value and a step whose 15th multiple passes bfloat16's range, as a group of values near both ends has."""
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: True)
    for one in (True, False) if dim == 128 else (False,):
        monkeypatch.setattr(ops, "_one_head_a_block", lambda *a: one)
        want, c = case(hq, hkv, dim, page).run().cpu(), case(hq, hkv, dim, page)
        rows = spoil(c, 3, 0, 280, 1, 0, -3.38e38)
        page_of, place = c.cache.tables[0][280 // page], 280 % page
        c.cache.pools[3][page_of, 1, place, 0] = 4.6e37
        c.cache.pools[2][page_of, 1, place] = 0xff
        got = c.run().cpu()
        hit = torch.zeros(len(c.q), hq, dtype=torch.bool)
        hit[:, hq // hkv:2 * hq // hkv] = rows.view(-1, 1)
        assert rows.any() and torch.equal(got[~hit], want[~hit])
