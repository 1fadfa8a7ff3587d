"""Attention over a cache of 4 bits whose block tables name pages that are none in the middle of sequences: their keys are not seen."""
import pytest
import torch
from cache4 import on
from cache4_sharp import beyond, expected, pages_hidden
from test_attention_cache4 import Case

from pulsar_b200 import ops

cuda = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


def with_holes(case, holes):
    """The case's table with pages {sequence: logical pages} that are none: -1 and the first id beyond the pool in turn."""
    table = case.table()
    for i, pages in holes.items():
        for j, p in enumerate(pages):
            table[i, p] = -1 if j % 2 == 0 else case.cache.pools[0].shape[0]
    return table


def check(case, holes):
    got = case.run(block_table=with_holes(case, holes).cuda()).cpu()
    want, most = expected(case.cache, case.q, case.q_lens, case.scale, case.window, pages_hidden(case.cache, holes))
    assert beyond(got, want, most) == 0, float((got.double() - want).abs().max())
    return got


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("page", [5, 8, 24, 16])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 64), (6, 3, 96), (4, 1, 128)])
def test_holes_far_into_a_sequence(dtype, page, hq, hkv, dim):
    """In turns that are otherwise seen whole, the third of a warp and later ones; a sequence without any beside them."""
    lens = [1500, 40, 1111]
    holes = {0: [3, 600 // page, 601 // page + 1, 900 // page, 1499 // page], 2: [700 // page, 1000 // page]}
    check(Case(lens, hq, hkv, dim, page, dtype, page + dim), holes)
    check(Case(lens, hq, hkv, dim, page, dtype, page + dim, window=950), {0: [800 // page, 1200 // page], 2: [700 // page]})


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("page", [5, 8, 24, 16])
def test_holes_that_portions_meet_on_codes(dtype, page, monkeypatch):
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: False)
    lens, q_lens = [1500, 40, 1111, 600], [9, 3, 1, 70]
    holes = {0: [600 // page, 1000 // page, 1495 // page], 2: [700 // page], 3: [520 // page, 560 // page]}
    check(Case(lens, 8, 2, 64, page, dtype, 50 + page, q_lens), holes)
    check(Case(lens, 6, 2, 96, page, dtype, 60 + page, q_lens, window=1000), holes)


@cuda
@pytest.mark.parametrize("page", [4, 16])
def test_a_sequence_of_holes_alone_gives_zeros(page):
    c = Case([700, 300], 8, 2, 64, page, torch.bfloat16, 70)
    table = c.table()
    table[0] = -1
    got = c.run(block_table=table.cuda())
    assert (got[0] == 0).all() and torch.equal(got[1], c.run()[1])
    short = c.run(block_table=table.cuda(), kv_len=on([0, 300]))
    assert torch.equal(short, got)
