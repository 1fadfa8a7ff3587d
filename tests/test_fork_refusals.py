"""Forks that cannot be, whatever refuses them: nothing is left behind.  And what a child may do where its parent ended."""
import pytest
import torch

from host_engine import HostEngine
from pulsar_b200 import ops
from pulsar_b200.cache import CacheError, CacheManager, CacheNeed
from pulsar_b200.engine.scheduler import SchedulerError


def rule(token, position):
    return (3 * token + position) % 500


def started(n=37, **kw):
    eng = HostEngine(rule, **kw)
    sid = eng.create_session(list(range(n)))
    eng.feed(sid, [], 6)
    while eng.has_work():
        eng.step(1)
    return eng, sid


def state(eng):
    return (eng.cache.n_free_pages(), eng.cache.n_free_slots(), eng.cache.n_shared_pages(), sorted(map(str, eng.cache.live_requests())),
            sorted(eng._sessions), eng._next_id, sorted(map(str, eng.scheduler._known)))


@pytest.mark.parametrize("what", ["scheduler", "scheduler, second child", "seed", "length"])
def test_a_fork_that_is_refused_leaves_nothing_behind(monkeypatch, what):
    eng, sid = started()
    before = state(eng)
    overrides, length, error = [None, None, None], None, SchedulerError
    if what.startswith("scheduler"):
        inner, calls = eng.scheduler.fork_request, []

        def refuse(*args):
            calls.append(1)
            if len(calls) == (2 if "second" in what else 1):
                raise SchedulerError("refused")
            inner(*args)
        monkeypatch.setattr(eng.scheduler, "fork_request", refuse)
    elif what == "seed":
        overrides, error = [None, {"seed": 1 << 80}, None], (RuntimeError, OverflowError, ValueError)
    else:
        length, error = 60, CacheError
    with pytest.raises(error):
        eng._fork(sid, overrides, length, None)
    assert state(eng) == before
    eng.cache.check_consistency()
    monkeypatch.undo()
    children = eng._fork(sid, [None, None, None], None, None)
    assert eng.cache.n_shared_pages() == [2] and len(children) == 3
    for s in [sid, *children]:
        eng.release(s)
    assert eng.cache.n_free_pages() == [64] and eng.cache.n_free_slots() == 8


@pytest.mark.parametrize("length", [16, 17])
def test_a_cache_fork_whose_copy_fails_leaves_nothing_behind(monkeypatch, length):
    m = CacheManager([CacheNeed.paged_kv(1, 8), CacheNeed.state((3,))], 16, 12, 6, torch.float32, "cpu")
    m.open("a")
    m.append("a", length)

    def fail(*args):
        raise torch.cuda.OutOfMemoryError("no more memory")
    monkeypatch.setattr(ops, "copy_pages", fail)
    before = (m.n_free_pages(), m.n_free_slots(), m.live_requests(), m.n_shared_pages())
    with pytest.raises(torch.cuda.OutOfMemoryError):
        m.fork("a", ["b", "c"])
    assert (m.n_free_pages(), m.n_free_slots(), m.live_requests(), m.n_shared_pages()) == before
    m.check_consistency()


@pytest.mark.parametrize("lookahead", [False, True])
@pytest.mark.parametrize("generation", [1, 2])
def test_a_fork_of_a_sequence_that_ended_on_the_stop_token_needs_a_token_too(lookahead, generation):
    """However the parent was stepped: refused without tokens, and with one the child goes on as the parent does."""
    stop = rule(rule(rule(36, 36), 37), 38)
    eng = HostEngine(rule, eos_id=stop)
    sid = eng.create_session(list(range(37)))
    eng.feed(sid, [], 40)
    events = []
    while eng.has_work():
        events += eng.step(1, lookahead=lookahead)
    assert events[-1] == (sid, stop, True)
    child = sid
    for _ in range(generation):
        child = eng.fork(child)
    for s in (sid, child):
        with pytest.raises(ValueError, match="stop token"):
            eng.feed(s, [], 5)
    out = {sid: [], child: []}
    for s in out:
        eng.feed(s, [11], 5)
    while eng.has_work():
        for s, token, _ in eng.step(1, lookahead=lookahead):
            out[s].append(token)
    assert out[sid] == out[child] and len(out[sid]) == 5
    assert eng.scheduler.seqs[sid].tokens == eng.scheduler.seqs[child].tokens == [*range(37), rule(36, 36), rule(rule(36, 36), 37), stop, 11, *out[sid]]


@pytest.mark.parametrize("lookahead", [False, True])
def test_a_fork_of_a_sequence_that_spent_its_budget_goes_on_without_tokens(lookahead):
    eng = HostEngine(rule, eos_id=501)
    sid = eng.create_session(list(range(37)))
    eng.feed(sid, [], 6)
    while eng.has_work():
        eng.step(1, lookahead=lookahead)
    child = eng.fork(sid)
    out = {sid: [], child: []}
    for s in out:
        eng.feed(s, [], 4)
    while eng.has_work():
        for s, token, _ in eng.step(1, lookahead=lookahead):
            out[s].append(token)
    assert out[sid] == out[child] and len(out[sid]) == 4
