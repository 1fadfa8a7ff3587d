"""What expanded pages of a cache of 4 bits hold beside the cache, through the scratch buffers that the engine keeps from call to call."""
import functools
import types

import pytest
import torch
from cache4_sharp import beyond, expected
from test_attention_cache4 import Case

from pulsar_b200 import ops
from pulsar_b200.engine.runner import ModelRunner

cuda = pytest.mark.gpu


def kept_scratch(device):
    """A runner's scratch buffers, without the runner: (the function, what it holds)."""
    runner = types.SimpleNamespace(_scratch={}, _scratch_views={}, scratch_epoch=0, _capturing=False, device=torch.device(device))
    return functools.partial(ModelRunner.scratch, runner), runner._scratch


def held(buffers, tags=("attn4.k", "attn4.v")):
    return sum(b.numel() * b.element_size() for (tag, _), b in buffers.items() if tag in tags)


def test_rooms_that_grow_stay_within_the_room():
    """Every width that fits, in an order that grows and one that does not: keys and values of 2 bytes, half the room each."""
    room, per_page = 1 << 24, 2 * 16 * 128
    most = room // (4 * per_page)                                        # pages
    for widths in (range(1, most + 1, 7), (3, most // 2 + 1, most - 1, 5, most), (most - 3, 2, most)):
        scratch, buffers = kept_scratch("cpu")
        for width in widths:
            shape = (width, 2, 16, 128)
            for tag in ("attn4.k", "attn4.v"):
                got = ops._expanded_room(scratch, tag, shape, torch.bfloat16)
                assert got.shape == shape and got.is_contiguous()
            assert held(buffers) <= room
    scratch, buffers = kept_scratch("cpu")
    for width in (1, 700, 701, 1000, 1500):                              # one sequence's pages alone
        ops._expanded_room(scratch, "attn4.k", (width, 1, 16, 64), torch.bfloat16)
        assert held(buffers) < 2 * (2 * 1500 * 16 * 64)


@cuda
def test_calls_of_growing_width_stay_within_the_room(monkeypatch):
    per_page = 4 * 2 * 16 * 128
    room = 1 << 21                                                        # 128 pages of keys and values
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: True)
    monkeypatch.setattr(ops, "EXPANDED_ROOM_4BIT", room)
    scratch, buffers = kept_scratch("cuda")
    for lens, q_lens in (([300, 200], [60, 40]), ([470] * 3, [50, 9, 140]), ([640] * 4, [20] * 4), ([1000, 900, 10], [30, 140, 10]), ([2040, 5], [33, 5])):
        case = Case(lens, 8, 2, 128, 16, torch.bfloat16, sum(lens), q_lens)
        got = case.run(scratch=scratch).cpu()
        want, most = expected(case.cache, case.q, q_lens, case.scale, expanded=True)
        assert beyond(got, want, most) == 0 and 0 < held(buffers) <= room, (lens, held(buffers))
    assert room == 128 * per_page
