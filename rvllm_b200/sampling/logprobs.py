"""Log probabilities of tokens, as a program reads them: of the sampled ones beside generation, of given ones when a
prompt is scored.  (The reference has none; its sampler works on the host's copy of the logits,
src/sampler.rs:68-129.)"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Tuple

import torch


@dataclass(frozen=True)
class TokenLogprob:
    """Of one token under the model's distribution at its place (temperature 1, nothing filtered)."""
    token: int
    logprob: float
    rank: int                                   # 1: the most probable one
    entropy: float                              # of the distribution, in nats
    top: List[Tuple[int, float]] = field(default_factory=list)     # the most probable ids and their log probabilities


class LogprobReader:
    """Launches `ops.token_logprobs` and copies its results to the host without waiting; `read` is called when the copies
    are known to be done."""

    def __init__(self, ops, logits: torch.Tensor, tokens: torch.Tensor, top: int):
        results = (tokens,) + ops.token_logprobs(logits, tokens, top)
        if logits.is_cuda:
            self._host = [torch.empty(t.shape, dtype=t.dtype, pin_memory=True) for t in results]
            for host, t in zip(self._host, results):
                host.copy_(t, non_blocking=True)
        else:
            self._host = list(results)

    def read(self) -> List[TokenLogprob]:
        return [TokenLogprob(t, lp, rank, h, list(zip(ids, best)))
                for t, lp, rank, h, best, ids in zip(*(t.tolist() for t in self._host))]
