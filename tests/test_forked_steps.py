"""Steps of forked requests: where the packed arrays stand that captured steps read, and candidates again and again on one engine."""
import ctypes
import random

import pytest
import torch

import helpers
from helpers import TINY
from pulsar_b200 import host
from pulsar_b200.cache import CacheManager, CacheNeed


def packed(m, rids, sources=None):
    """A step of one token for each of ``rids``: the offsets of the packed arrays, and the arrays."""
    n, groups = len(rids), len(m.groups)
    ids, ones, zeros = host.longs([m.native_id(r, create=True) for r in rids]), host.ints([1] * n), host.ints([0] * n)
    src = host.ints(sources or [-1] * n)
    starts, slots, widths, bad = (ctypes.c_int * n)(), (ctypes.c_int * n)(), (ctypes.c_int * groups)(), ctypes.c_int()
    total = m._lib.ph_step_plan(m._h, n, ids, ones, zeros, ones, zeros, src, 64, 100, 64, starts, slots, widths, ctypes.byref(bad))
    assert total > 0
    buf, count = (ctypes.c_int * total)(), 7 + 2 * groups + (2 if sources else 0)
    offsets, lengths = (ctypes.c_int * count)(), (ctypes.c_int * count)()
    assert m._lib.ph_step_pack(m._h, n, ids, ones, zeros, ones, zeros, src, starts, slots, widths, ctypes.addressof(buf), total, offsets, lengths) == total
    spans = sorted((o, o + ln) for o, ln in zip(offsets, lengths))
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and spans[-1][1] <= total and all(o % 4 == 0 for o in offsets)
    return list(offsets), [list(buf[o:o + ln]) for o, ln in zip(offsets, lengths)], list(slots)


@pytest.mark.parametrize("groups", [1, 2, 3])
@pytest.mark.parametrize("children", [2, 4, 7])
@pytest.mark.parametrize("length", [3, 50, 65])
@pytest.mark.parametrize("device_tokens", [False, True])
def test_what_captured_steps_read_stands_still_whatever_the_tables_gain(groups, children, length, device_tokens):
    m = CacheManager([CacheNeed.paged_kv(2, 16, None if g == 0 else 20 * g) for g in range(groups)], 16, 400, 10)
    m.set_resident_tables(True)
    rids = [f"c{i}" for i in range(children)]
    for r in rids:
        m.open(r)
        m.append(r, length)
    packed(m, rids)
    sources = list(range(children)) if device_tokens else None
    steady, _, _ = packed(m, rids, sources)                 # nothing or one page gained
    for r in rids:
        m.close(r)
    m.open("a")
    m.append("a", length)
    m.fork("a", rids)
    read = [*range(7), *(7 + 2 * g for g in range(groups))]  # the tables themselves stand elsewhere, applied before the step
    for step in range(20):
        offsets, arrays, slots = packed(m, rids, sources)
        assert [offsets[k] for k in read] == [steady[k] for k in read], step
        for g in range(groups):
            assert arrays[7 + 2 * g] == [m.slots(r, g, length + step, 1)[0] for r in rids]
            count, *triples = arrays[8 + 2 * g]
            gained = [triples[3 * i:3 * i + 3] for i in range(count)]
            whole = [[slot, lp, page] for r, slot in zip(rids, slots) for lp, page in enumerate(m.table(r, g))]
            assert gained == (whole if step == 0 else [t for t in whole if t[1] * 16 == length + step])
        if device_tokens:
            assert arrays[-2] == list(range(children)) and arrays[-1] == sources


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "C", "E"])
def test_candidates_again_and_again_replay_captured_steps(tmp_path, name):
    """C and E have a second group of pages, behind a window: the first step of every set of forks brings whole tables."""
    from pulsar_b200.engine.engine import Engine
    raw, seed, page = TINY[name]
    folder = helpers.make_folder(tmp_path / "m", raw, seed)
    cfg = dict(dtype="float32", page_size=page, num_pages=200, max_sessions=12, max_running=12, max_chunk_size=64, eos_id=-1)
    plain, eng = Engine(folder, cfg), Engine(folder, cfg)
    eng.runner.SHARED_KEYS_SAVED = 1
    replays = []
    for i in range(4):
        prompt = helpers.random_tokens(random.Random(i), 41 + i, raw["vocab_size"])
        got = eng.candidates(prompt, 5, 14, temperature=0.9, top_k=40, seed=10 * i)
        want = plain.generate([prompt] * 5, 14, temperature=0.9, top_k=40, seed=10 * i)
        assert sorted(c.tokens for c in got) == sorted(want), i
        replays.append(eng.runner.graph_replays)
    assert replays[0] > 0 and replays[3] > replays[2] > replays[1] > replays[0]
    eng.cache.check_consistency()
