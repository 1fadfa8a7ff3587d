"""Continuations of one prompt beside one another, and beside other sequences: pages that run short, events, scores."""
import random

import pytest

import helpers
from helpers import TINY
from host_engine import HostEngine


def rule(token, position):
    return (7 * token + position) % 900


def alone(prompt, n):
    out, last = [], prompt[-1]
    for p in range(len(prompt) - 1, len(prompt) - 1 + n):
        last = rule(last, p)
        out.append(last)
    return out


@pytest.mark.parametrize("pages", [16, 19, 26, 34, 60])
def test_continuations_finish_where_pages_run_short(pages):
    """Four of 70 tokens behind 160: 15 pages each by themselves.  One that lost its pages gets them from those that are over."""
    prompt = list(range(160))
    eng = HostEngine(rule, num_pages=pages)
    got = eng.candidates(prompt, 4, 70)
    assert [c.tokens for c in got] == [alone(prompt, 70)] * 4
    assert all([s.token for s in c.scores] == c.tokens and [s.logprob for s in c.scores] == [-float(t) for t in c.tokens] for c in got)
    assert (eng.scheduler.n_preemptions > 0) == (pages < 34)
    assert not eng._sessions and not eng.has_work() and eng.cache.n_free_pages() == [pages] and eng.cache.n_free_slots() == 8
    eng.cache.check_consistency()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "C"])
def test_a_continuation_that_lost_its_pages_is_what_it_would_have_been(tmp_path, name):
    from pulsar_b200.engine.engine import Engine
    raw, seed, page = TINY[name]
    folder = helpers.make_folder(tmp_path / "m", raw, seed)
    cfg = dict(dtype="float32", page_size=page, max_sessions=8, max_running=8, max_chunk_size=64, eos_id=-1)
    prompt = helpers.random_tokens(random.Random(4), 5 * page + 3, raw["vocab_size"])
    new = 6 * page
    eng = Engine(folder, dict(cfg, num_pages=20))
    got = eng.candidates(prompt, 4, new, temperature=0.9, top_k=40, seed=5)
    want = Engine(folder, dict(cfg, num_pages=80)).generate([prompt] * 4, new, temperature=0.9, top_k=40, seed=5)
    assert sorted(c.tokens for c in got) == sorted(want) and eng.scheduler.n_preemptions > 0
    assert all(len(c.scores) == new for c in got) and not eng._sessions
    eng.cache.check_consistency()


@pytest.mark.parametrize("lookahead", [False, True])
def test_other_sequences_events_reach_the_next_step(lookahead):
    """A scored sequence that runs beside two sets of candidates: every token is an event of ``step`` once and in order, and its score comes with it."""
    eng = HostEngine(rule)
    sid = eng.create_session(list(range(20)), scores=0)
    eng.feed(sid, [], 25)
    got, scored = [], []

    def take(events):
        got.extend(tok for s, tok, _ in events if s == sid)
        scored.extend(eng.scores(sid))
        assert [s.token for s in scored] == got
    for _ in range(4):
        take(eng.step(1, lookahead=lookahead))
    for prompt in (list(range(30, 70)), [5, 6, 7]):
        before = len(got)
        assert [c.tokens for c in eng.candidates(prompt, 3, 6)] == [alone(prompt, 6)] * 3
        assert eng.scores(sid) == [] and not eng._mailbox
        take(eng.step(1, lookahead=lookahead))
        assert len(got) > before + 5
    while eng.has_work():
        take(eng.step(1, lookahead=lookahead))
    assert got == alone(list(range(20)), 25) and eng.session_state(sid) == "parked"


def test_events_of_others_outlive_an_exception_between():
    eng = HostEngine(rule, num_pages=12)
    sid = eng.create_session(list(range(20)))
    eng.feed(sid, [], 25)
    inner, passes = eng._launch, []

    def launch(plan):
        passes.append(1)
        if len(passes) == 9:
            raise RuntimeError("a pass that could not be launched")
        return inner(plan)
    eng._launch = launch
    with pytest.raises(RuntimeError, match="launched"):
        eng.candidates([1, 2, 3], 2, 20)
    eng._launch = inner
    got = []
    while eng.has_work():
        got += [tok for s, tok, _ in eng.step(1) if s == sid]
    assert got == alone(list(range(20)), 25)
    assert sorted(eng._sessions) == [sid]
