"""Requests that share pages: the cache's accounting (forked, given back, moved into pools of another size), families, the scheduler; and on a GPU
the engine's forks, candidates and scores against runs of their own and against the plain implementation."""
import random

import pytest
import torch

import helpers
from helpers import TINY, TOL
from pulsar_b200.cache import CacheError, CacheManager, CacheNeed, OutOfPages
from pulsar_b200.engine.scheduler import Scheduler, SchedulerError

cuda = pytest.mark.gpu


def manager(pages=12, page=4, window=None, max_requests=6, state=False):
    needs = [CacheNeed.paged_kv(2, 16), CacheNeed.paged_kv(2, 16)]
    if window is not None:
        needs.append(CacheNeed.paged_kv(2, 16, window))
    if state:
        needs.append(CacheNeed.state((3,)))
    return CacheManager(needs, page, pages, max_requests)


# ------------------------------------------------------------------------------------------------ accounting
@pytest.mark.parametrize("length", [0, 1, 3, 4, 5, 8, 9, 10])
def test_a_fork_shares_whole_pages_and_has_the_rest_for_itself(length):
    m = manager()
    m.open("a")
    m.append("a", 10)                                   # pages 0, 1, 2
    m.fork("a", ["b", "c"], length)
    whole, rest = divmod(length, 4)
    for child in ("b", "c"):
        assert m.length(child) == length and m.table(child, 0)[:whole] == [0, 1, 2][:whole] and len(m.table(child, 0)) == whole + bool(rest)
    if rest:
        own = {m.table("b", 0)[whole], m.table("c", 0)[whole]}
        assert len(own) == 2 and not own & {0, 1, 2}
    assert [m.page_holders(0, p) for p in range(3)] == [3 if p < whole else 1 for p in range(3)] and m.n_shared_pages() == [whole]
    assert m.n_free_pages() == [12 - 3 - 2 * bool(rest)]
    m.check_consistency()
    m.close("a")                                        # what the children share stays
    m.check_consistency()
    assert m.n_free_pages() == [12 - whole - 2 * bool(rest)] and m.n_shared_pages() == [whole]
    assert m.append("b", 3) == length
    m.close("c")
    m.check_consistency()
    assert m.n_shared_pages() == [0]
    m.close("b")
    assert m.n_free_pages() == [12] and m.n_free_slots() == 6


def test_a_fork_of_a_fork_and_families():
    m = manager(pages=30, max_requests=9)
    m.open("a")
    m.append("a", 17)
    m.fork("a", ["b"])
    m.append("b", 6)                                    # 23 tokens
    m.fork("b", ["c", "d"], 20)
    m.open("x")
    m.append("x", 9)
    m.fork("x", ["y"], 8)
    m.open("z")
    m.append("z", 5)
    assert m.page_holders(0, 0) == 4 and m.page_holders(0, m.table("b", 0)[4]) == 3
    families, shared = m.families(["y", "d", "z", "a", "x", "c"], 0)
    assert families == [[0, 4], [1, 3, 5]] and shared == [8, 16, 0, 16, 8, 16]        # of a, c and d: what all three have
    assert m.families(["c", "d"], 0) == ([[0, 1]], [20, 20])
    assert m.families(["a", "z", "x"], 0) == ([], [0, 0, 0]) and m.families([], 0) == ([], [])
    m.check_consistency()


def test_a_fork_that_cannot_be_changes_nothing():
    m = manager(pages=4, max_requests=3)
    m.open("a")
    m.append("a", 10)
    before = (m.n_free_pages(), m.n_free_slots(), m.live_requests(), m.n_shared_pages())
    for error, args, said in ((OutOfPages, ("a", ["b", "c"]), "page each"), (OutOfPages, ("a", ["b", "c", "d"], 8), "state slots"), (CacheError, ("a", ["b"], 11), "cannot be forked"),
                              (CacheError, ("a", ["b"], -1), "cannot be forked"), (CacheError, ("q", ["b"]), "unknown"), (CacheError, ("a", ["a"]), "already open"),
                              (CacheError, ("a", ["b", "b"], 8), "already open")):
        with pytest.raises(error, match=said):
            m.fork(*args)
        assert (m.n_free_pages(), m.n_free_slots(), m.live_requests(), m.n_shared_pages()) == before
        m.check_consistency()
    m.fork("a", [])
    m.fork("a", ["b", "c"], 8)
    m.check_consistency()


def test_fixed_size_state_is_forked_at_its_length_only():
    m = manager(state=True)
    m.open("a")
    m.append("a", 6)
    with pytest.raises(CacheError, match="fixed-size state"):
        m.fork("a", ["b"], 4)
    m.fork("a", ["b"])
    assert m.state_slot("b") != m.state_slot("a")


def test_windows_give_back_shared_pages_with_their_last_holder():
    m = manager(pages=20, window=6)
    m.open("a")
    m.append("a", 8)
    m.fork("a", ["b"])
    assert m.n_shared_pages() == [2, 2]
    m.append("a", 8)                                    # the query at 16 sees keys from 11 on
    m.release_passed("a")
    assert m.table("a", 1)[:2] == [-1, -1] and m.table("b", 1)[:2] == [0, 1] and m.page_holders(1, 0) == 1
    assert m.reclaimable("b") == [0, 0]
    m.append("b", 4)
    assert m.release_passed("b") >= 1 and m.page_holders(1, 0) == 0
    m.check_consistency()
    with pytest.raises(CacheError, match="released page"):
        m.fork("a", ["c"], 9)                           # the query at 9 would see keys from 4 on, which are gone
    assert not m.has("c")
    m.fork("a", ["c"])
    m.append("c", 1)
    m.check_consistency()
    for r in ("a", "b", "c"):
        m.close(r)
    assert m.n_free_pages() == [20, 20]
    m.check_consistency()


def test_pages_that_others_hold_do_not_count_as_reclaimable():
    m = manager(pages=9, window=4)
    m.open("a")
    m.append("a", 16)
    m.fork("a", ["b"])
    assert m.reclaimable("a") == [0, 0]                 # the window has passed three pages, b holds them too
    m.close("b")
    assert m.reclaimable("a")[1] == 3


@pytest.mark.parametrize("pages", [5, 6, 9, 40])
def test_pools_of_another_size(pages):
    m = manager(pages=16)
    for r, n in (("a", 3), ("b", 9), ("c", 4)):
        m.open(r)
        m.append(r, n)
    m.close("a")
    m.fork("b", ["d"], 8)
    m.fork("b", ["e"])
    m.close("c")
    before = {r: m.table(r, 0) for r in ("b", "d", "e")}
    ids = sorted(set(sum(before.values(), [])))
    assert len(ids) == 4
    m.resize(pages)
    for r, table in before.items():
        assert m.table(r, 0) == [ids.index(p) for p in table]
    assert m.n_free_pages() == [pages - 4] and m.groups[0].allocator.n == pages and m.page_holders(0, ids.index(before["b"][0])) == 3
    m.check_consistency()
    m.append("d", min(5, (pages - 4) * 4))
    m.check_consistency()
    for r in ("b", "d", "e"):
        m.close(r)
    assert m.n_free_pages() == [pages]


def test_pools_too_small_are_refused():
    m = manager(pages=8, window=100)
    m.open("a")
    m.append("a", 13)
    for bad in (3, [4, 3], [4], 0, -1):
        with pytest.raises(CacheError if bad in ([4], 0, -1) else OutOfPages):
            m.resize(bad)
        assert m.n_free_pages() == [4, 4]
    m.resize([4, 7])
    assert m.n_free_pages() == [0, 3]


@pytest.mark.parametrize("seed", range(6))
def test_random_forks_appends_releases_and_resizes(seed):
    rng = random.Random(seed)
    m = manager(pages=40, window=9 if seed % 2 else None, max_requests=8)
    live, n = [], 0
    for _ in range(400):
        what = rng.random()
        try:
            if what < 0.2 or not live:
                m.open(n)
                live.append(n)
                n += 1
            elif what < 0.5:
                m.append(rng.choice(live), rng.randint(1, 7))
            elif what < 0.7:
                r = rng.choice(live)
                m.fork(r, [n, n + 1][:rng.randint(1, 2)], None if rng.random() < 0.5 else rng.randint(0, m.length(r)))
                live += [c for c in (n, n + 1) if m.has(c)]
                n += 2
            elif what < 0.85:
                m.close(live.pop(rng.randrange(len(live))))
            elif what < 0.9:
                m.release_passed(rng.choice(live))
            else:
                m.resize(rng.randint(20, 60))
        except (OutOfPages, CacheError):
            pass
        m.check_consistency()
    for r in live:
        m.close(r)
    assert m.n_free_pages() == [g.allocator.n for g in m.groups] and m.n_shared_pages() == [0] * len(m.groups)


def test_the_scheduler_runs_a_forked_request_from_where_it_begins():
    m = manager(pages=20)
    s = Scheduler(m, 4, 16)

    def step():
        plan = s.schedule()
        for e in plan:
            if not m.has(e.rid):
                m.open(e.rid)
            m.append(e.rid, len(e.tokens))
        s.on_step(plan)
        return plan
    s.add_request("a", [1, 2, 3, 4, 5, 6], 2)
    assert [e.tokens for e in step()] == [[1, 2, 3, 4, 5, 6]]
    s.on_token("a", 7, -1)
    s.park("a")
    m.fork("a", ["b"], 5)
    s.fork_request("a", "b", 5)
    with pytest.raises(SchedulerError, match="already known"):
        s.fork_request("a", "b", 5)
    with pytest.raises(SchedulerError, match="not all cached"):
        s.fork_request("a", "c", 7)
    assert not s.has_work() and s.seqs["b"].tokens == [1, 2, 3, 4, 5] and s.seqs["b"].n_cached == 5
    s.extend_request("b", [9, 8], 3)
    assert [(e.rid, e.tokens, e.sample) for e in step()] == [("b", [9, 8], True)]
    assert m.length("b") == 7 and m.table("b", 0)[0] == m.table("a", 0)[0]
    m.check_consistency()
    s.finish("a")
    s.finish("b")
    assert m.n_free_pages() == [20]


# ------------------------------------------------------------------------------------------------ the engine
@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for name in ("A", "C", "E", "F"):
        raw, seed, _ = TINY[name]
        d = tmp_path_factory.mktemp(f"fork{name}")
        helpers.make_folder(d, raw, seed)
        out[name] = str(d)
    return out


def engine(folder, dtype, page, **kw):
    from pulsar_b200.engine.engine import Engine
    cfg = dict(dtype=dtype, page_size=page, num_pages=200, max_sessions=12, max_running=12, max_chunk_size=64, eos_id=-1)
    cfg.update(kw)
    return Engine(folder, cfg)


@cuda
@pytest.mark.parametrize("name", ["A", "C", "E", "F"])
@pytest.mark.parametrize("n_prompt", [1, 2, 16, 17, 45])
def test_candidates_are_what_sessions_of_their_own_generate(folders, name, n_prompt):
    """float32, so that the ways of the attention differ in last bits only: the tokens are the same, and their scores those of the plain
    implementation's logits."""
    raw, seed, page = TINY[name]
    eng = engine(folders[name], "float32", page)
    eng.runner.SHARED_KEYS_SAVED = 1                     # the attention over shared pages wherever there are any
    prompt = helpers.random_tokens(random.Random(n_prompt), n_prompt, raw["vocab_size"])
    got = eng.candidates(prompt, 5, 12, temperature=0.9, top_k=40, seed=100, alternatives=3)
    assert eng.cache.live_requests() == [] and all(f == 200 for f in eng.cache.n_free_pages()) and not eng._sessions
    want = engine(folders[name], "float32", page).generate([prompt] * 5, 12, temperature=0.9, top_k=40, seed=100)
    assert sorted(c.tokens for c in got) == sorted(want)
    assert [c.mean_logprob for c in got] == sorted((c.mean_logprob for c in got), reverse=True)
    cfg, weights = helpers.read_folder(folders[name])
    for c in got:
        logits = helpers.plain_logits(cfg, weights, prompt + c.tokens)[n_prompt - 1:-1].double()
        log_p = torch.log_softmax(logits, 1)
        near = 3 * TOL["float32"] * float(logits.abs().max())
        for i, s in enumerate(c.scores):
            assert s.token == c.tokens[i] and abs(s.logprob - float(log_p[i, s.token])) < near
            assert abs(s.entropy + float((log_p[i].exp() * log_p[i]).sum())) < near * 8
            assert len(s.alternatives) == 3 and abs(s.alternatives[0][1] - float(log_p[i].max())) < near
            assert abs(s.rank - int((log_p[i] > log_p[i, s.token]).sum())) <= int(((log_p[i] - log_p[i, s.token]).abs() < near).sum())


@cuda
@pytest.mark.parametrize("name,tokens", [("E", 200), ("F", 300)])
def test_forked_steps_on_the_tensor_cores_follow_the_plain_logits(folders, name, tokens):
    """bfloat16 with heads of 128 (tcgen05) and 64: the captured steps of eight forks, their logits against the plain implementation's."""
    raw, seed, page = TINY[name]
    cfg, weights = helpers.read_folder(folders[name])
    w16 = helpers.as_bf16_matrices(weights)
    eng = engine(folders[name], "bfloat16", page, num_pages=400)
    eng.runner.SHARED_KEYS_SAVED = 1
    used = []
    from pulsar_b200 import ops
    inner = ops.paged_attention_shared
    try:
        ops.paged_attention_shared = lambda *a, **k: (used.append(1), inner(*a, **k))
        prompt = helpers.random_tokens(random.Random(5), tokens, raw["vocab_size"])
        got = eng.candidates(prompt, 8, 10, temperature=1.0, seed=7)
    finally:
        ops.paged_attention_shared = inner
    assert used and eng.runner.graph_replays > 0
    for c in got[:3]:
        logits = helpers.plain_logits(cfg, w16, prompt + c.tokens)[tokens - 1:-1].double()
        log_p = torch.log_softmax(logits, 1)
        near = 2 * TOL["bfloat16"] * float(logits.abs().max())
        assert all(abs(s.logprob - float(log_p[i, s.token])) < near for i, s in enumerate(c.scores))


@cuda
def test_forks_of_sessions_go_on_from_where_they_stand(folders):
    raw, seed, page = TINY["A"]
    eng = engine(folders["A"], "float32", page)
    prompt = helpers.random_tokens(random.Random(1), 21, raw["vocab_size"])
    a = eng.create_session(prompt)
    eng.feed(a, [], 6)
    tokens = {a: []}
    eng._run_turns(tokens)
    b, c = eng.fork(a, scores=2), eng.fork(a, length=16)
    assert eng.session_state(b) == "parked" and eng.cache.n_shared_pages() == [1]
    eng.feed(a, [], 5)
    eng.feed(b, [], 5)                                   # greedy as the parent: the same tokens
    eng.feed(c, prompt[16:], 6)
    more = {a: [], b: [], c: []}
    eng._run_turns(more)
    assert more[a] == more[b] and more[c] == tokens[a] and len(eng.scores(b)) == 5 and eng.scores(b) == []
    eng.release(a)
    assert [len(p) for p in eng.context_pages(b)][0] == page
    with pytest.raises(ValueError, match="without scores"):
        eng.scores(c)
    for sid in (b, c):
        eng.release(sid)
    assert all(f == 200 for f in eng.cache.n_free_pages())
    eng.cache.check_consistency()


@cuda
def test_scores_come_in_order_however_steps_overlap(folders):
    raw, seed, page = TINY["F"]
    prompts = [helpers.random_tokens(random.Random(i), 5 + 9 * i, raw["vocab_size"]) for i in range(4)]
    runs = []
    for lookahead in (False, True):
        eng = engine(folders["F"], "float32", page)
        ids = [eng.create_session(p, {"temperature": 0.8, "seed": i}, scores=i if i < 3 else None) for i, p in enumerate(prompts)]
        for sid in ids:
            eng.feed(sid, [], 7)
        out = {sid: [] for sid in ids}
        while eng.has_work():
            for sid, tok, _ in eng.step(1, lookahead=lookahead):
                out[sid].append(tok)
        runs.append([(out[s], eng.scores(s) if i < 3 else None) for i, s in enumerate(ids)])
        for i, s in enumerate(ids[:3]):
            assert [x.token for x in runs[-1][i][1]] == out[s] and all(len(x.alternatives) == i for x in runs[-1][i][1])
    assert [[t for t, _ in r] for r in runs][0] == [[t for t, _ in r] for r in runs][1]
    for (_, x), (_, y) in zip(*runs):
        assert x is None or all(abs(p.logprob - q.logprob) < 1e-4 and p.rank == q.rank for p, q in zip(x, y))


@cuda
@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("C", "float32"), ("E", "bfloat16"), ("F", "bfloat16")])
def test_scored_prompts(folders, name, dtype):
    raw, seed, page = TINY[name]
    cfg, weights = helpers.read_folder(folders[name])
    eng = engine(folders[name], dtype, page, max_chunk_size=31)
    prompts = [helpers.random_tokens(random.Random(n), n, raw["vocab_size"]) for n in (1, 2, 31, 33, 80)]
    bare, whole = eng.score(prompts), eng.score(prompts, alternatives=4)
    assert [len(r) for r in bare] == [len(p) - 1 for p in prompts] and eng.cache.live_requests() == []
    for p, x, y in zip(prompts, bare, whole):
        if len(p) < 2:
            continue
        logits = helpers.plain_logits(cfg, helpers.as_bf16_matrices(weights) if dtype == "bfloat16" else weights, p)[:-1].double()
        log_p = torch.log_softmax(logits, 1)
        near = 2 * TOL[dtype] * float(logits.abs().max())
        for i, (a, b) in enumerate(zip(x, y)):
            assert a.token == b.token == p[i + 1] and abs(a.logprob - float(log_p[i, p[i + 1]])) < near and abs(a.logprob - b.logprob) < 1e-4
            assert abs(a.entropy - b.entropy) < 1e-4 and a.rank is None and len(b.alternatives) == 4
            assert b.rank >= 4 or b.alternatives[b.rank] == (b.token, b.logprob)


@cuda
def test_a_cache_of_another_size_in_mid_turn(folders):
    raw, seed, page = TINY["A"]
    prompts = [helpers.random_tokens(random.Random(n), 20 + n, raw["vocab_size"]) for n in range(3)]
    want = engine(folders["A"], "float32", page).generate(prompts, 30)
    eng = engine(folders["A"], "float32", page)
    ids = [eng.create_session(p) for p in prompts]
    for sid in ids:
        eng.feed(sid, [], 30)
    out = {sid: [] for sid in ids}
    sizes = iter([14, 300, 13])
    for turn in range(200):
        if turn in (4, 9, 15):
            eng.resize_cache(next(sizes))
            eng.cache.check_consistency()
        for sid, tok, _ in eng.step(1):
            out[sid].append(tok)
        if not eng.has_work():
            break
    assert [out[s] for s in ids] == want and eng.cache.groups[0].pools["k"].shape[1] == 13
    with pytest.raises(ValueError, match="do not hold"):
        eng.resize_cache(2)
    with pytest.raises(OutOfPages):
        eng.resize_cache(8)
    for sid in ids:
        eng.release(sid)
    assert eng.cache.n_free_pages() == [13]


@cuda
def test_refusals_of_the_engine(folders):
    raw, seed, page = TINY["A"]
    eng = engine(folders["A"], "float32", page, max_sessions=4, max_running=4)
    with pytest.raises(RuntimeError, match="sessions"):
        eng.candidates([1, 2, 3], 4, 5)
    with pytest.raises(ValueError, match="at least one token"):
        eng.candidates([], 2, 5)
    with pytest.raises(ValueError, match="at least one token"):
        eng.candidates([1], 0, 5)
    with pytest.raises(ValueError, match="alternatives"):
        eng.candidates([1, 2], 2, 5, alternatives=33)
    with pytest.raises(ValueError, match="alternatives"):
        eng.create_session([1], scores=-1)
    with pytest.raises(ValueError, match="vocabulary"):
        eng.score([[1, 2, 100000]])
    s = eng.create_session([1, 2, 3])
    with pytest.raises(ValueError, match="nothing in the cache"):
        eng.fork(s)
    eng.feed(s, [], 3)
    with pytest.raises(RuntimeError, match="still generating"):
        eng.fork(s)
    while eng.has_work():
        eng.step(1)
    with pytest.raises(CacheError, match="cannot be forked"):
        eng.fork(s, length=50)
    with pytest.raises(ValueError, match="override"):
        eng.fork(s, {"warmth": 1})
    assert not any(eng._sessions[x].state == "active" for x in eng._sessions) and len(eng._sessions) == 1
    eng.release(s)
    assert len(eng.candidates([5, 6, 7, 8], 3, 4)) == 3 and all(f == 200 for f in eng.cache.n_free_pages())


@cuda
@pytest.mark.parametrize("model", ["bubotar A", "bubotar S", "bosenex A"])
def test_models_with_fixed_size_state_fork_it(tmp_path, model):
    """The states of recurrent layers are copied (S: there is nothing but states): the continuations are those of sessions of their own."""
    import copy

    import test_bosenex
    import test_bubotar
    raw = copy.deepcopy((test_bubotar if model.startswith("bubotar") else test_bosenex).CONFIGS[model[-1]][0])
    folder = helpers.make_folder(tmp_path / "m", raw, 3, store_dtype=torch.bfloat16)
    kw = dict(num_pages=64, max_sessions=6, max_running=6, max_chunk_size=256)
    prompt = helpers.random_tokens(random.Random(2), 27, raw["vocab"])
    got = engine(folder, "float32", 16, **kw).candidates(prompt, 4, 8, temperature=0.8, seed=3)
    want = engine(folder, "float32", 16, **kw).generate([prompt] * 4, 8, temperature=0.8, seed=3)
    assert sorted(c.tokens for c in got) == sorted(want)


@cuda
def test_command_line_candidates(folders, capsys):
    import json
    from pulsar_b200 import cli
    args = ["--model", folders["A"], "--dtype", "float32", "--prompt_ids", "1,2,3,4,5", "--prompt_ids", "9,8", "--gen_tokens", "6", "--temperature", "0.8",
            "--seed", "4", "--candidates", "3", "--eos_id", "-1", "--active_buffer_size", "256", "--json"]
    assert cli.main(args) == 0
    found = json.loads(capsys.readouterr().out)
    assert len(found["outputs"]) == len(found["mean_logprobs"]) == 6 and all(len(o) == 6 for o in found["outputs"])
    assert found["mean_logprobs"][:3] == sorted(found["mean_logprobs"][:3], reverse=True)
