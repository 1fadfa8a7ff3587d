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


def both_ways(monkeypatch, case, holes):
    """The way on codes and the one over expanded pages, with one and two heads a block where it has both: what sequences without holes get does not change."""
    for expanded, one in ((False, False), (True, False), (True, True)):
        monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: expanded)
        monkeypatch.setattr(ops, "_one_head_a_block", lambda *a: one and case.cache.dim == 128)
        whole = case.run().cpu()
        got = case.run(block_table=with_holes(case, holes).cuda()).cpu()
        want, most = expected(case.cache, case.q, case.q_lens, case.scale, case.window, pages_hidden(case.cache, holes), expanded)
        _, on_codes = expected(case.cache, case.q, case.q_lens, case.scale, case.window, pages_hidden(case.cache, holes))
        at = 0
        for i, count in enumerate(case.q_lens):
            if holes.get(i):                            # taken on codes
                most[at:at + count] = on_codes[at:at + count]
            else:
                assert torch.equal(got[at:at + count], whole[at:at + count])
            at += count
        assert beyond(got, want, most) == 0, (expanded, one, float((got.double() - want).abs().max()))


@cuda
@pytest.mark.parametrize("window", [None, 300])
@pytest.mark.parametrize("hq,hkv,dim,page", [(8, 2, 128, 16), (3, 3, 128, 8), (32, 4, 64, 4), (8, 2, 64, 16), (4, 2, 128, 64)])
def test_holes_that_portions_meet_either_way(monkeypatch, hq, hkv, dim, page, window):
    lens, q_lens = [700, 40, 333, 0, 520, 300], [150, 40, 1, 0, 200, 260]
    c = Case(lens, hq, hkv, dim, page, torch.bfloat16, 80 + page, q_lens, window=window)
    both_ways(monkeypatch, c, {0: [470 // page, 480 // page + 1, 699 // page], 4: [500 // page], 5: [0, 128 // page, 299 // page]})


@cuda
def test_holes_that_no_query_sees_change_nothing(monkeypatch):
    """Behind the last key, before the window."""
    c = Case([700, 130], 8, 2, 128, 16, torch.bfloat16, 90, [100, 130], window=64)
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: True)
    table = c.cache.table(width=60)
    want = c.run(block_table=table.cuda())
    table[0, :33], table[0, 44:], table[1, 9:] = -1, -1, 1 << 30
    assert torch.equal(c.run(block_table=table.cuda()), want)


@cuda
def test_holes_in_runs_of_sequences_and_in_a_captured_call(monkeypatch):
    lens, q_lens = [400, 130, 0, 390, 64, 100, 40], [300, 130, 0, 260, 0, 100, 33]
    c = Case(lens, 8, 2, 128, 16, torch.bfloat16, 91, q_lens)
    monkeypatch.setattr(ops, "EXPANDED_ROOM_4BIT", 2 * 4 * 25 * 2 * 16 * 128)
    holes = {0: [3, 10], 3: [20], 5: [0]}
    both_ways(monkeypatch, c, holes)
    args = c.args(block_table=with_holes(c, holes).cuda())
    ops.paged_attention_4bit(**args)
    want = args["out"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention_4bit(**args)
    args["out"].zero_()
    args["block_table"].copy_(c.table())                 # the lengths and tables that a replay finds are the ones that count
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(args["out"], c.run())
    args["block_table"].copy_(with_holes(c, holes))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(args["out"], want)


@cuda
def test_many_sequences_under_a_wide_table(monkeypatch):
    """One long portion among 250, a table of 131,072 keys: more turns than the kernel on codes can deal out, which a look for holes does not do."""
    lens, q_lens = [2000] + [3 + i % 20 for i in range(249)], [2000] + [1 + i % 3 for i in range(249)]
    c = Case(lens, 8, 1, 64, 16, torch.bfloat16, 92, q_lens)
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: True)
    holes = {0: [5, 60], 7: [0]}
    wide = torch.full((len(lens), 8192), -1, dtype=torch.int32)
    table = with_holes(c, holes)
    wide[:, :table.shape[1]] = table
    got = c.run(block_table=wide.cuda()).cpu()
    want, most = expected(c.cache, c.q, q_lens, c.scale, None, pages_hidden(c.cache, holes), True)
    _, on_codes = expected(c.cache, c.q, q_lens, c.scale, None, pages_hidden(c.cache, holes))
    assert beyond(got, want, torch.maximum(most, on_codes)) == 0
