"""Pools of another size: every group moves or none does, whatever fails on the way."""
import random

import pytest
import torch

import helpers
from helpers import TINY
from pulsar_b200 import ops
from pulsar_b200.cache import CacheManager, CacheNeed


def plain_copy(src_pools, dst_pools, src, dst):
    for a, b in zip(src_pools, dst_pools):
        b[:, dst.long()] = a[:, src.long()]


def filled(window=5):
    """Two groups of two entries; every position of every request holds a number of its own."""
    m = CacheManager([CacheNeed.paged_kv(1, 8), CacheNeed.paged_kv(1, 8, window), CacheNeed.paged_kv(1, 8), CacheNeed.paged_kv(1, 8, window)], 4, 10, 5, torch.float32, "cpu")
    for r, n in (("a", 6), ("b", 9), ("c", 3)):
        m.open(r)
        m.append(r, n)
    m.close("a")                                             # the held pages are not the first ones
    m.fork("b", ["d"], 8)
    for i, r in enumerate(("b", "c")):
        for entry in range(4):
            pools = m.pools(entry)
            for p, slot in enumerate(m.slots(r, m.group_of_entry[entry], 0, m.length(r))):
                for k, name in enumerate(pools):
                    pools[name].view(-1, 8)[slot] = 1000 * entry + 100 * i + 10 * k + p
    return m


def seen(m):
    """What a step would read: for every request and entry its keys and values through table and pools."""
    out = {}
    for r in ("b", "c", "d"):
        for entry in range(4):
            slots = m.slots(r, m.group_of_entry[entry], 0, m.length(r))
            out[r, entry] = [pool.view(-1, 8)[slots].tolist() for pool in m.pools(entry).values()]
    return out


def accounts(m):
    return [m.n_free_pages(), [m.table(r, g) for r in ("b", "c", "d") for g in range(2)], m.n_shared_pages(), [g.allocator.n for g in m.groups]]


@pytest.mark.parametrize("size", [5, 8, 40, [30, 6]])
def test_every_group_moves(monkeypatch, size):
    monkeypatch.setattr(ops, "copy_pages", plain_copy)
    m = filled()
    before = seen(m)
    m.resident_table(0, 3)
    m.resize(size)
    m.check_consistency()
    sizes = size if isinstance(size, list) else [size, size]
    assert seen(m) == before and [g.allocator.n for g in m.groups] == sizes and not m.resident
    assert [m.pools(e)["k"].shape[0] for e in (0, 1)] == sizes == [g.pools["k"].shape[1] for g in m.groups]
    assert m.append("b", 1) == 9


# four pools are asked for, then two copies, one group behind the other
@pytest.mark.parametrize("what", ["zeros", "copy"])
@pytest.mark.parametrize("at", range(4))
def test_a_failure_on_the_way_changes_nothing(monkeypatch, what, at):
    m = filled()
    before, kept, pools = seen(m), accounts(m), [dict(g.pools) for g in m.groups]
    calls = []

    def failing(inner):
        def call(*args, **kw):
            calls.append(1)
            if len(calls) == at + 1:
                raise torch.cuda.OutOfMemoryError("no more memory")
            return inner(*args, **kw)
        return call
    monkeypatch.setattr(ops, "copy_pages", failing(plain_copy) if what == "copy" else plain_copy)
    if what == "zeros":
        monkeypatch.setattr(torch, "zeros", failing(torch.zeros))
    if what == "copy" and at >= 2:
        m.resize(30)                                         # there are two copies only
        assert seen(m) == before
        return
    with pytest.raises(torch.cuda.OutOfMemoryError):
        m.resize(30)
    monkeypatch.undo()
    m.check_consistency()
    assert accounts(m) == kept and seen(m) == before
    assert all(g.pools[name] is p[name] for g, p in zip(m.groups, pools) for name in p)
    assert all(m.pools(e)["k"].data_ptr() == m.groups[m.group_of_entry[e]].pools["k"][m.index_in_group[e]].data_ptr() for e in range(4))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["C", "E"])
def test_a_resize_that_fails_in_mid_turn_leaves_the_sequences_as_they_were(tmp_path, monkeypatch, name):
    """Models with two groups: the second group's memory cannot be had, then it can; captured steps before, between and after."""
    from pulsar_b200.engine.engine import Engine
    raw, seed, page = TINY[name]
    folder = helpers.make_folder(tmp_path / "m", raw, seed)
    cfg = dict(dtype="float32", page_size=page, num_pages=120, max_sessions=4, max_running=4, max_chunk_size=64, eos_id=-1)
    prompts = [helpers.random_tokens(random.Random(n), 20 + n, raw["vocab_size"]) for n in range(3)]
    want = Engine(folder, cfg).generate(prompts, 40)
    eng = Engine(folder, cfg)
    ids = [eng.create_session(p) for p in prompts]
    for sid in ids:
        eng.feed(sid, [], 40)
    out = {sid: [] for sid in ids}
    zeros, calls = torch.zeros, []

    def once(*args, **kw):
        calls.append(1)
        if len(calls) == 3:                                  # the second group's first pool
            raise torch.cuda.OutOfMemoryError("no more memory")
        return zeros(*args, **kw)
    for turn in range(200):
        if turn == 10:
            with monkeypatch.context() as m:
                m.setattr(torch, "zeros", once)
                with pytest.raises(torch.cuda.OutOfMemoryError):
                    eng.resize_cache(300)
            assert [g.pools["k"].shape[1] for g in eng.cache.groups] == [120, 120] and eng.config.num_pages == 120
        if turn == 20:
            eng.resize_cache(200)
        for sid, tok, _ in eng.step(1):
            out[sid].append(tok)
        if not eng.has_work():
            break
    assert [out[s] for s in ids] == want and eng.runner.graph_replays > 0
    assert [g.pools["k"].shape[1] for g in eng.cache.groups] == [200, 200]
    eng.cache.check_consistency()
