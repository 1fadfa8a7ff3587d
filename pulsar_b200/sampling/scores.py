"""What a step's logits say of the tokens that were taken from them, as the engine hands it to its users."""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Tuple

import torch

from .. import ops


@dataclass
class TokenScore:
    """A token's log probability (natural logarithm, of the logits as they are: no temperature, no filter), how many tokens were likelier, the
    entropy of what could have come, and the likeliest tokens with their log probabilities, in order.  ``rank`` is None where only the
    first two were asked for (``Engine.score`` without alternatives)."""
    token: int
    logprob: float
    entropy: float
    rank: Optional[int] = None
    alternatives: List[Tuple[int, float]] = field(default_factory=list)


@dataclass
class Candidate:
    """One of several continuations of a prompt, with the score of each of its tokens."""
    tokens: List[int]
    scores: List[TokenScore]

    @property
    def logprob(self) -> float:
        """Of the whole continuation."""
        return sum(s.logprob for s in self.scores)

    @property
    def mean_logprob(self) -> float:
        return self.logprob / max(1, len(self.scores))


class ScoreBoard:
    """Device memory for the scores of up to ``rows`` tokens with ``top`` alternatives each, one run of 32-bit words, so that one copy brings
    them to the host: log probabilities, entropies, ranks [rows], then the alternatives' ids and log probabilities [rows, top]."""

    def __init__(self, rows: int, top: int, device):
        self.rows, self.top = rows, top
        self.words = torch.empty(rows * (3 + 2 * top), dtype=torch.float32, device=device)

    @staticmethod
    def n_words(rows: int, top: int) -> int:
        return rows * (3 + 2 * top)

    def take(self, logits: torch.Tensor, tokens: torch.Tensor) -> None:
        """Score ``tokens`` (int32 [rows]) by ``logits`` [rows, vocab], in the stream."""
        r, n = self.rows, self.top
        parts = self.words.split([r, r, r, r * n, r * n])
        ids, logprobs = (parts[3].view(torch.int32).view(r, n), parts[4].view(r, n)) if n else (None, None)
        ops.token_scores(logits, tokens, parts[0], parts[1], parts[2].view(torch.int32), ids, logprobs)

    @staticmethod
    def read(host: torch.Tensor, rows: int, top: int, tokens: List[int]) -> List[TokenScore]:
        """The scores from the words on the host (float32)."""
        logprob, entropy, rank, ids, logprobs = host[:ScoreBoard.n_words(rows, top)].split([rows, rows, rows, rows * top, rows * top])
        rank, ids = rank.view(torch.int32).tolist(), ids.view(torch.int32).tolist()
        logprob, entropy, logprobs = logprob.tolist(), entropy.tolist(), logprobs.tolist()
        return [TokenScore(int(t), logprob[i], entropy[i], rank[i], list(zip(ids[i * top:(i + 1) * top], logprobs[i * top:(i + 1) * top])))
                for i, t in enumerate(tokens)]
