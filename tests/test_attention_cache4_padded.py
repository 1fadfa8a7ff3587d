"""Portions over a cache of 4 bits with more tokens than keys, as a padded batch has them: queries before the first key see nothing and give zeros."""
import pytest
import torch
from cache4_sharp import beyond, expected
from test_attention_cache4 import Case

from pulsar_b200 import ops

cuda = pytest.mark.gpu


def check(case, expanded):
    got = case.run().cpu()
    want, most = expected(case.cache, case.q, case.q_lens, case.scale, case.window, expanded=expanded)
    assert beyond(got, want, most) == 0
    at = 0
    for n, count in zip(case.cache.lens, case.q_lens):
        assert (got[at:at + max(0, count - n)] == 0).all()
        at += count


@cuda
@pytest.mark.parametrize("expanded", [False, True])
@pytest.mark.parametrize("window", [None, 60])
@pytest.mark.parametrize("lens,q_lens", [([400, 0, 130, 0], [300, 400, 130, 5]), ([50, 300], [600, 40]), ([0, 0], [256, 129]), ([1], [129]), ([127, 5], [128, 300])])
@pytest.mark.parametrize("hq,hkv,dim,page", [(8, 2, 128, 16), (3, 1, 128, 16), (8, 2, 64, 8), (4, 4, 128, 64)])
def test_portions_of_more_tokens_than_keys(monkeypatch, expanded, window, lens, q_lens, hq, hkv, dim, page):
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: expanded)
    for one in (True, False) if expanded and dim == 128 else (False,):
        monkeypatch.setattr(ops, "_one_head_a_block", lambda *a: one)
        check(Case(lens, hq, hkv, dim, page, torch.bfloat16, sum(lens) + page, q_lens, window=window), expanded)


@cuda
@pytest.mark.parametrize("lens,q_lens", [([0, 200], [300, 100]), ([50], [600])])
def test_portions_of_more_tokens_than_keys_in_float32(lens, q_lens):
    check(Case(lens, 8, 2, 128, 16, torch.float32, 3, q_lens), False)
