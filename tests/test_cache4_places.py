"""Pools of a cache of 4 bits where a layer's part of a cache's pool starts: steps of few groups in small pages start at multiples of 4 and 8 bytes."""
import random

import pytest
import torch
from cache4 import on
from test_attention_cache4 import Case
from test_cache4 import Rows

import helpers
from pulsar_b200 import ops

cuda = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


def moved(pool, nbytes):
    """The pool's contents ``nbytes`` behind a multiple of 16 bytes."""
    room = torch.empty(pool.numel() * pool.element_size() + 64, dtype=torch.uint8, device="cuda")
    at = (-room.data_ptr()) % 16 + nbytes
    got = room[at:at + pool.numel() * pool.element_size()].view(pool.dtype).view(pool.shape)
    got.copy_(pool)
    assert got.data_ptr() % 16 == nbytes % 16
    return got


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim,page,least", [(32, 1, 4), (32, 5, 4), (96, 3, 4), (224, 2, 4), (64, 1, 8), (64, 8, 8), (192, 24, 8), (160, 7, 4)])
def test_steps_at_places_of_rows(dtype, dim, page, least):
    """All three operators give the same bits as with pools that start at multiples of 16 bytes, and refuse places between rows."""
    for nbytes in (least, 16 - least):
        r = Rows(9, 4, 2, dim, page, dtype, seed=dim + page)
        for x, y in zip(r.run(), r.run(k_steps=moved(r.pools[1], nbytes), v_steps=moved(r.pools[3], nbytes))):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        for q_lens in (None, [60, 17, 3]):
            c = Case([200, 17, 40], 4, 2, dim, page, dtype, dim, q_lens)
            steps = dict(k_steps=moved(c.cache.pools[1], nbytes), v_steps=moved(c.cache.pools[3], nbytes))
            assert torch.equal(c.run(), c.run(**steps))
        table = c.table().cuda()
        got = []
        for where in (dict(k_steps=c.cache.pools[1].cuda(), v_steps=c.cache.pools[3].cuda()), steps):
            out = [torch.zeros(table.numel(), 2, page, dim, dtype=dtype, device="cuda") for _ in range(2)]
            ops.expand_pages_4bit(c.cache.pools[0].cuda(), where["k_steps"], c.cache.pools[2].cuda(), where["v_steps"], table, on(c.cache.lens), *out, torch.empty_like(table))
            got.append(out)
        assert all(torch.equal(a, b) for a, b in zip(*got))
    for run, pools in ((r.run, r.pools), (c.run, c.cache.pools)):
        with pytest.raises(ops.KernelError, match=f"multiple of {least} bytes"):
            run(k_steps=moved(pools[1], 2))
    with pytest.raises(ops.KernelError, match=f"multiple of {least} bytes"):
        ops.expand_pages_4bit(c.cache.pools[0].cuda(), moved(c.cache.pools[1], 2), c.cache.pools[2].cuda(), c.cache.pools[3].cuda(), table, on(c.cache.lens), *out, torch.empty_like(table))


@cuda
def test_steps_of_pages_of_16_start_at_multiples_of_16_bytes():
    c = Case([40], 4, 2, 32, 16, torch.bfloat16, 3)
    with pytest.raises(ops.KernelError, match="multiple of 16 bytes"):
        c.run(v_steps=moved(c.cache.pools[3], 8))


@cuda
@pytest.mark.parametrize("page,pages", [(1, 197), (3, 67), (5, 41)])
def test_an_engine_whose_layers_start_between_multiples_of_16_bytes(tmp_path, page, pages):
    """Two heads of 32 in three layers: a layer's steps take pages * page * 8 bytes."""
    from pulsar_b200.engine.engine import Engine
    raw, seed, usual = helpers.TINY["B"]
    folder = helpers.make_folder(tmp_path, raw, seed)
    prompts = [helpers.random_tokens(random.Random(5), n, raw["vocab_size"]) for n in (30, 70)]

    def tokens(page, pages):
        return Engine(folder, dict(dtype="float32", page_size=page, num_pages=pages, max_sessions=4, max_running=4, max_chunk_size=64, eos_id=-1, cache_bits=4)).generate(prompts, 12)
    assert page * pages * 8 % 16 == 8 and tokens(page, pages) == tokens(usual, 64)
