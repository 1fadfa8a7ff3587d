"""Captured steps of forked sequences: prompts of many lengths share them, and no more than a bounded number is kept."""
import random

import pytest

import helpers
from helpers import TINY
from pulsar_b200 import ops
from pulsar_b200.engine.runner import ModelRunner


def test_the_ones_used_last_are_kept():
    runner = object.__new__(ModelRunner)
    runner._graphs, runner._graph_seen, runner.MOST_SHARED_GRAPHS = {}, {}, 3
    other = [(n, n, n, (64,), False, (), (1,)) for n in range(20)]
    shared = [(n, n, n, (64,), False, ((0, 2, n, 1024, 512),), (1,)) for n in range(6)]
    for k in other + shared:
        runner._graph_seen[k] = 3
    for k in other:
        runner._keep_graph(k, ())
    for k in shared[:3]:
        runner._keep_graph(k, ())
    runner._graphs[shared[0]] = runner._graphs.pop(shared[0])            # used again
    for k in shared[3:5]:
        runner._keep_graph(k, ())
    assert [k for k in runner._graphs if k[5]] == [shared[0], *shared[3:5]] and all(k in runner._graphs for k in other)
    assert set(runner._graph_seen) == {*other, shared[0], *shared[3:]}                # 5 was never kept


def test_longer_shared_keys_than_the_rounding_says_are_cut_alike(monkeypatch):
    monkeypatch.setattr(ops, "fn", lambda name: lambda dtype, rows, d, page: 16 if rows <= 16 or d != 128 else 128)
    for families, members, hq, hkv, dim in ((1, 2, 32, 8, 128), (1, 32, 32, 8, 128), (3, 8, 4, 1, 64), (1, 40, 1, 1, 96)):
        cut = [ops.shared_cut.__wrapped__(families * members, families, members, keys, 512, hq, hkv, dim, 16, ops.torch.bfloat16)
               for keys in (ops.SHARED_CUT_KEYS, ops.SHARED_CUT_KEYS + 1, 10 * ops.SHARED_CUT_KEYS)]
        assert cut[0] == cut[1] == cut[2]


@pytest.mark.gpu
def test_prompts_of_many_lengths_find_the_same_captured_steps(tmp_path):
    """Page 8, tables in steps of 64 pages: lengths of 300 to 480 differ in nothing that a captured step depends on.  And sets of two to seven with
    room for two captured steps."""
    from pulsar_b200.engine.engine import Engine
    raw, seed, page = TINY["E"]
    folder = helpers.make_folder(tmp_path / "m", raw, seed)
    cfg = dict(dtype="float32", page_size=page, num_pages=600, max_sessions=12, max_running=12, max_chunk_size=512, eos_id=-1)
    plain, eng = Engine(folder, cfg), Engine(folder, cfg)
    eng.runner.SHARED_KEYS_SAVED = 1
    kept = []
    for i, length in enumerate((300, 333, 401, 480, 355, 417)):
        prompt = helpers.random_tokens(random.Random(length), length, raw["vocab_size"])
        got = eng.candidates(prompt, 4, 9, temperature=0.9, top_k=40, seed=i)
        assert sorted(c.tokens for c in got) == sorted(plain.generate([prompt] * 4, 9, temperature=0.9, top_k=40, seed=i))
        kept.append([k for k in eng.runner._graphs if k[5]])
    assert len(kept[0]) == 1 and kept[-1] == kept[0]
    eng.runner.MOST_SHARED_GRAPHS = 2
    for n in range(2, 8):
        prompt = helpers.random_tokens(random.Random(n), 60 + n, raw["vocab_size"])
        got = eng.candidates(prompt, n, 9, temperature=0.9, top_k=40, seed=n)
        assert sorted(c.tokens for c in got) == sorted(plain.generate([prompt] * n, 9, temperature=0.9, top_k=40, seed=n))
        assert len([k for k in eng.runner._graphs if k[5]]) <= 2


@pytest.mark.parametrize("heads,dim,page,dtype,keys", [(8, 128, 16, "bfloat16", 24576), (8, 64, 16, "bfloat16", 24576), (2, 128, 16, "bfloat16", 49152), (1, 64, 16, "bfloat16", 196608),
                                                       (1, 64, 16, "float32", 24576), (1, 96, 16, "bfloat16", 24576), (1, 64, 4, "bfloat16", 24576)])
def test_small_keys_have_to_be_more(heads, dim, page, dtype, keys):
    """On the tensor cores 48 MiB of keys and values that need not be read, wherever a key and its value are less than 2 KB."""
    import torch
    from pulsar_b200.cache import CacheManager, CacheNeed
    runner = object.__new__(ModelRunner)
    runner.cache = CacheManager([CacheNeed.paged_kv(heads, dim)], page, 4, 2, getattr(torch, dtype), "cpu")
    assert runner._least_saved(0) == keys
    runner.SHARED_KEYS_SAVED = 1
    assert runner._least_saved(0) == keys // 24576
