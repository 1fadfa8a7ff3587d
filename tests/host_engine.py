"""The engine's host side alone: sessions, scheduler, page accounting and the booking of passes, with a rule in the place of the model."""
from types import SimpleNamespace

import torch

from pulsar_b200.cache import CacheManager, CacheNeed
from pulsar_b200.config.engine_config import EngineConfig
from pulsar_b200.engine.engine import Engine, _Inflight
from pulsar_b200.engine.scheduler import UNREAD, Scheduler
from pulsar_b200.sampling.sampler import Sampler
from pulsar_b200.sampling.scores import ScoreBoard


class HostEngine(Engine):
    """``rule(token, position)`` is what a pass samples behind a token at a position; its log probability is minus the token it samples."""

    def __init__(self, rule, needs=None, vocab=1000, **config):
        cfg = dict(page_size=16, num_pages=64, max_sessions=8, max_running=8, max_chunk_size=512, eos_id=-1)
        cfg.update(config)
        self.rule, self.config, self.eos_id = rule, EngineConfig.from_dict(cfg), cfg["eos_id"]
        c = self.config
        self.model = SimpleNamespace(spec=SimpleNamespace(vocab_size=vocab))
        self.cache = CacheManager(needs or [CacheNeed.paged_kv(2, 16)], c.page_size, c.num_pages, c.max_sessions)
        self.runner = SimpleNamespace(forget_addresses=lambda: None)
        self.scheduler = Scheduler(self.cache, c.max_running, c.max_chunk_size)
        self._sessions, self._next_id, self.forwards, self._mailbox, self._inflight, self._unclaimed, self._failed = {}, 0, 0, {}, None, [], None

    def _launch(self, plan):
        before, last, at = self._inflight, {}, {}
        for e in plan:
            tokens = list(e.tokens)
            if tokens[-1] == UNREAD:
                tokens = [before.report.host[Sampler.HEAD + before.row_of[e.rid]].item()]
            if not self.cache.has(e.rid):
                self.cache.open(e.rid)
            self.cache.release_passed(e.rid)
            at[e.rid] = self.cache.append(e.rid, len(tokens)) + len(tokens) - 1
            last[e.rid] = tokens[-1]
        self.forwards += 1
        self.scheduler.on_step(plan)
        sampled = [e.rid for e in plan if e.sample]
        ids = [self.rule(last[r], at[r]) for r in sampled]
        report = SimpleNamespace(wait=lambda: None, host=torch.tensor([0] * Sampler.HEAD + ids, dtype=torch.int32))
        sessions = [self._sessions[r] for r in sampled]
        top = max((s.alternatives for s in sessions if s.alternatives is not None), default=None)
        scores = None
        if top is not None:
            words = torch.zeros(ScoreBoard.n_words(len(ids), top))
            words[:len(ids)] = -torch.tensor(ids, dtype=torch.float32)
            scores = (SimpleNamespace(host=words), top)
        for r in sampled:
            self.scheduler.on_sampled(r)
        return _Inflight(sampled, {r: i for i, r in enumerate(sampled)}, report, [0.0 if s.params.greedy else s.draw() for s in sessions], scores)
