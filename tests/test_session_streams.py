"""Sessions that stream beside one another: every token once, in order, with its score, whoever stepped the engine."""
import random

import pytest

from host_engine import HostEngine
from pulsar_b200.api import Session


def rule(token, position):
    return (5 * token + position) % 700


def alone(prompt, n):
    out, last = [], prompt[-1]
    for p in range(len(prompt) - 1, len(prompt) - 1 + n):
        last = rule(last, p)
        out.append(last)
    return out


def opened(eng, lengths, n):
    prompts = [list(range(10 * i, 10 * i + length)) for i, length in enumerate(lengths)]
    sessions = [Session(eng.create_session(p, scores=0), eng) for p in prompts]
    for s in sessions:
        s.send([], n)
    return prompts, sessions


def test_one_session_behind_the_other():
    """The second one's turn is over before anybody reads it."""
    prompts, sessions = opened(HostEngine(rule), (5, 9, 2), 7)
    for p, s in zip(prompts, sessions):
        assert list(s.recv()) == alone(p, 7)
        assert [x.token for x in s.scores()] == alone(p, 7) and s.scores() == []


@pytest.mark.parametrize("seed", range(5))
def test_tokens_taken_in_turns(seed):
    prompts, sessions = opened(HostEngine(rule), (5, 9, 2, 30), 11)
    rng, streams, got, scored = random.Random(seed), [s.recv() for s in sessions], [[] for _ in sessions], [[] for _ in sessions]
    live = list(range(4))
    while live:
        i = rng.choice(live)
        for _ in range(rng.randint(1, 4)):
            tok = next(streams[i], None)
            if tok is None:
                live.remove(i)
                break
            got[i].append(tok)
            scored[i] += [x.token for x in sessions[i].scores()]
            assert scored[i] == got[i]
    assert got == [alone(p, 11) for p in prompts]


def test_a_stream_beside_candidates_and_steps():
    eng = HostEngine(rule)
    prompts, (a, b) = opened(eng, (5, 9), 30)
    stream = a.recv()
    got = [next(stream) for _ in range(3)]
    eng.candidates([1, 2, 3], 3, 5)
    got += list(stream)
    assert got == alone(prompts[0], 30) and list(b.recv()) == alone(prompts[1], 30)
