"""The engine with keys and values in 4 bits: against the plain decoder whose attention reads quantised keys and values, and what sessions do with pages."""
import math
import random

import pytest
import torch
from cache4 import Cache4, attended, bound, quantised

import helpers
from helpers import TINY
from plain import qwen3_plain as plain

cuda = pytest.mark.gpu
NAMES = ["B", "D", "E"]                       # heads of 32, 64 (a window), 128 (a window)

# Beside the bars of a cache in the dtype (helpers.TOL): a value whose code lies next to a border may fall on its other side, one step (about 0.27
# of a standard deviation, as the largest and least of 32 lie 4.1 of them apart) off.  float32 activations are off by some 1e-6 of that: a border is
# that near for one value in 1e5, of the ten thousands that these requests cache, and one step more or less in one element of a key or value moves
# an output by less than a hundredth.  bfloat16 activations reach the cache through two roundings of 2^-8, and so does the least value of their
# group, 2.05 standard deviations from zero, from which codes count: together (0.8 + 2.05) 2^-7 = 0.022, 8 in a hundred of a step.  As many codes
# fall the other way, which adds sqrt(0.08) * 0.27 = 0.077 standard deviations to every key and value.  The first positions of a request have
# nothing that would average this out: their attention's output is off by as much, in each of the two or three layers, sqrt(3) * 0.077 = 0.13.
BAR = {"float32": 1e-2, "bfloat16": 2e-2 + 0.13}


def kept(x, dtype):
    """What a cache of 4 bits makes of float64 heads [T, H, D] that a cache of ``dtype`` would hold rounded."""
    codes, step, least = quantised(x.to(dtype).double())
    return (least.unsqueeze(-1) + step.unsqueeze(-1) * codes).flatten(-2)


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for name in NAMES:
        raw, seed, _ = TINY[name]
        out[name] = str(helpers.make_folder(tmp_path_factory.mktemp(f"four{name}"), raw, seed))
    return out


def plain_rows(folder, dtype, requests, monkeypatch):
    """Plain logits of every request, with keys and values as a cache of 4 bits keeps them."""
    exact = plain.attention
    kind = torch.float32 if dtype == "float32" else torch.bfloat16
    monkeypatch.setattr(plain, "attention", lambda q, k, v, scale, window=None: exact(q, kept(k, kind), kept(v, kind), scale, window))
    cfg, weights = helpers.read_folder(folder)
    weights = helpers.as_bf16_matrices(weights) if dtype == "bfloat16" else weights
    return {rid: helpers.plain_logits(cfg, weights, tokens) for rid, tokens in requests.items()}


@cuda
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("shape", ["whole", "tail", "portions", "mixed"])
def test_logits(folders, monkeypatch, name, dtype, shape):
    from pulsar_b200.replay import Replay
    raw, seed, page = TINY[name]
    rng = random.Random(seed + 5)
    requests = {r: helpers.random_tokens(rng, n, raw["vocab_size"]) for r, n in (("a", 190), ("b", 47), ("c", 75), ("d", 21))}
    if shape == "mixed":
        trace = helpers.trace_mixed(requests, rng, portion=(2, 60))
    else:
        requests = {"a": requests["a"]}
        trace = {"whole": helpers.trace_whole, "tail": helpers.trace_tail, "portions": lambda t: helpers.trace_portions(t, [70, 3, 40, 2])}[shape](requests["a"])
    want = plain_rows(folders[name], dtype, requests, monkeypatch)
    replay = Replay(folders[name], dtype, 4096, page, cache_bits=4)
    worst = 0.0
    for record, rows in zip(trace.records, trace.rows):
        got = replay.run_step(record)
        for row, (rid, pos) in enumerate(rows):
            worst = max(worst, float((got[row].double() - want[rid][pos]).abs().max() / want[rid].abs().max()))
    assert helpers.report(f"cache4.{name}.{shape}", worst, dtype) < BAR[dtype]


@cuda
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", NAMES)
def test_every_attention_of_mixed_steps(folders, monkeypatch, name, dtype):
    """Each call that the steps make, from the pages it is given, against the formula in 64 bits."""
    from pulsar_b200 import ops
    from pulsar_b200.replay import Replay
    raw, seed, page = TINY[name]
    rng = random.Random(seed + 6)
    requests = {r: helpers.random_tokens(rng, n, raw["vocab_size"]) for r, n in (("a", 150), ("b", 20), ("c", 60))}
    trace = helpers.trace_mixed(requests, rng, portion=(20, 70))
    run, calls = ops.paged_attention_4bit, []

    def checked(q, k, ks, v, vs, out, table, kv_len, scale, window=None, cu_q=None, q_lens=None, scratch=None):
        run(q, k, ks, v, vs, out, table, kv_len, scale, window, cu_q, q_lens, scratch)
        lens = kv_len.tolist()
        cache = Cache4([], k.shape[1], q.shape[2], k.shape[2], 0)
        cache.lens, cache.pools = lens, [t.cpu() for t in (k, ks, v, vs)]
        cache.tables = [[max(p, 0) for p in row[:-(-n // cache.page)]] for row, n in zip(table.tolist(), lens)]
        first = 0 if cu_q is None else int(cu_q[0])
        counts = [1] * len(lens) if q_lens is None else q_lens
        rows = slice(first, first + sum(counts))
        want, score_size, value_size = attended(cache, q[rows].cpu(), counts, scale, window)
        off, most = (out[rows].cpu().double() - want).abs(), bound(want, score_size, value_size, q.dtype, max(lens))
        assert (off <= most).all(), (float(off.max()), float(most.max()))
        calls.append((cu_q is not None, max(counts)))

    monkeypatch.setattr(ops, "paged_attention_4bit", checked)
    replay = Replay(folders[name], dtype, 4096, page, cache_bits=4)
    replay.runner.cuda_graphs = False
    for record in trace.records:
        replay.run_step(record)
    assert any(portions for portions, _ in calls) and any(not portions for portions, _ in calls) and max(n for _, n in calls) > 20


def engine(folder, page, **more):
    from pulsar_b200.engine.engine import Engine
    return Engine(folder, dict(dict(dtype="bfloat16", page_size=page, num_pages=256, max_sessions=8, max_running=8, max_chunk_size=64, eos_id=-1, cache_bits=4), **more))


@cuda
@pytest.mark.parametrize("name", NAMES)
def test_captured_steps_give_the_same_tokens(folders, name):
    raw, _, page = TINY[name]
    rng = random.Random(1)
    prompts = [helpers.random_tokens(rng, n, raw["vocab_size"]) for n in (30, 100, 5)]
    eager, captured = engine(folders[name], page, cuda_graphs=False), engine(folders[name], page)
    want = eager.generate(prompts, 40)
    assert captured.generate(prompts, 40) == want and captured.runner.graph_replays > 0 and eager.runner.graph_replays == 0
    assert captured.cache.live_requests() == []


@cuda
def test_the_command_line_and_the_python_entry_point(folders, capsys):
    import json

    from pulsar_b200 import cli
    from pulsar_b200.api import Pulsar
    raw, _, page = TINY["D"]
    prompt = helpers.random_tokens(random.Random(3), 70, raw["vocab_size"])
    want = engine(folders["D"], page).generate([prompt], 8)[0]
    args = ["--model", folders["D"], "--prompt_ids", ",".join(map(str, prompt)), "--gen_tokens", "8", "--dtype", "bfloat16", "--page_size", str(page), "--max_pages", "64",
            "--eos_id", "-1", "--cache_bits", "4", "--json"]
    assert cli.main(args) == 0
    assert json.loads(capsys.readouterr().out)["outputs"] == [want]
    p = Pulsar(folders["D"], dict(page_size=page, num_pages=64, max_sessions=4, max_running=4, eos_id=-1, cache_bits=4))
    assert {t.dtype for g in p.engine.cache.groups for t in g.pools.values()} == {torch.uint8, torch.bfloat16}
    s = p.create_session(prompt[:50])
    s.send(prompt[50:], 8)
    assert list(s.recv()) == want


@cuda
def test_forked_sequences_go_on_as_their_parent(folders):
    """A fork in the middle of a page: the children's greedy tokens are the parent's, on pages shared and copied in 4 bits."""
    raw, _, page = TINY["D"]
    eng = engine(folders["D"], page)
    prompt = helpers.random_tokens(random.Random(2), 3 * page + 5, raw["vocab_size"])
    alone = eng.generate([prompt], 12)[0]
    sid = eng.create_session(prompt)
    eng.feed(sid, [], 4)
    first = []
    while eng.has_work():
        first += [tok for s, tok, _ in eng.step(1) if s == sid]
    assert first == alone[:4]
    kids = [eng.fork(sid) for _ in range(3)]
    got = {k: [] for k in kids}
    for k in kids:
        eng.feed(k, [], 8)
    while eng.has_work():
        for s, tok, _ in eng.step(1):
            got[s].append(tok)
    assert got[kids[0]] == got[kids[1]] == got[kids[2]] and got[kids[0]][:2] == alone[4:6]
    eng.cache.check_consistency()


@cuda
def test_pools_of_another_size_hold_the_same(folders):
    raw, _, page = TINY["E"]
    prompt = helpers.random_tokens(random.Random(3), 70, raw["vocab_size"])
    want = engine(folders["E"], page).generate([prompt], 20)[0]
    eng = engine(folders["E"], page)
    sid = eng.create_session(prompt)
    eng.feed(sid, [], 10)
    got = []
    while eng.has_work():
        got += [tok for _, tok, _ in eng.step(1)]
    eng.resize_cache(64)
    eng.feed(sid, [], 10)
    while eng.has_work():
        got += [tok for _, tok, _ in eng.step(1)]
    assert got == want


@cuda
def test_a_text_is_scored(folders):
    raw, _, page = TINY["D"]
    text = helpers.random_tokens(random.Random(4), 60, raw["vocab_size"])
    scores = engine(folders["D"], page).score([text])[0]
    assert len(scores) in (59, 60) and all(math.isfinite(s.logprob) and s.logprob <= 0 for s in scores[1:])


def test_a_token_takes_three_tenths_of_the_memory():
    from pulsar_b200.config import config_from_dict
    from pulsar_b200.models import build_model
    for dtype, share in ((torch.bfloat16, 5 / 16), (torch.float32, 5 / 32)):
        whole, four = (build_model(config_from_dict(helpers.TINY_E), dtype, bits).cache_needs()[0].bytes_per_token(dtype) for bits in (0, 4))
        assert four == share * whole


def test_what_has_no_cache_of_4_bits_is_refused():
    from pulsar_b200.config import EngineConfig, config_from_dict
    from pulsar_b200.config.model_config import ConfigError
    from pulsar_b200.models import build_model
    with pytest.raises(ConfigError, match="multiple of 32"):
        build_model(config_from_dict(helpers.TINY_A), torch.float32, 4)                     # heads of 16
    with pytest.raises(ConfigError, match="at most 256"):
        build_model(config_from_dict(dict(helpers.TINY_B, head_dim=288)), torch.float32, 4)
    with pytest.raises(ConfigError, match="0 .* or 4"):
        EngineConfig.from_dict(dict(cache_bits=8))
    with pytest.raises(ConfigError, match="in 4 bits, found 2"):
        build_model(config_from_dict(helpers.TINY_B), torch.float32, 2)
    assert build_model(config_from_dict(helpers.TINY_B), torch.float32, 4).cache_bits == 4 and build_model(config_from_dict(helpers.TINY_B), torch.float32).cache_bits == 0


def test_designs_with_other_mixers_are_refused():
    from pulsar_b200.config.model_config import ConfigError
    from pulsar_b200.config.registry import config_from_dict
    from pulsar_b200.models import build_model
    from test_megusun import MEGU_A
    from test_topunex import TOPU_C
    with pytest.raises(ConfigError, match="cache_bits=4: mixers .* have no cache"):
        build_model(config_from_dict(MEGU_A), torch.bfloat16, 4)                            # recurrences
    with pytest.raises(ConfigError, match="cache_bits=4: .* dense form"):
        build_model(config_from_dict(TOPU_C), torch.bfloat16, 4)                            # caps, sinks and gates
