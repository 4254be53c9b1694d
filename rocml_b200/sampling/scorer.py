"""Log probabilities of tokens, with the rows' entropy and most likely tokens, on the GPU.

One kernel reads the logits once (csrc/logprobs.cu); a few numbers a row come back to the host.  As with sampling, ``launch`` enqueues and
``collect`` waits, through a ring of pinned buffers.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

from .. import kernels


@dataclass
class TokenScore:
    """A token's natural log probability where it stands, the entropy of the distribution it was one of, and that distribution's most
    likely tokens with theirs, most likely first.  The distribution is the softmax of the logits, before temperature, top-k and top-p."""

    token: int
    logprob: float
    entropy: float
    top: List[Tuple[int, float]]


@dataclass
class PendingScores:
    n: int
    top: int
    host: torch.Tensor
    event: "torch.cuda.Event"


class Scorer:
    def __init__(self, device, max_batch: int, depth: int = 4):
        self.device = torch.device(device)
        self.max_batch = max_batch
        self._rings = {}           # top -> pinned buffers, made when they are first asked for
        self._depth = depth

    def launch(self, logits: torch.Tensor, tokens: torch.Tensor, top: int) -> PendingScores:
        """Score ``tokens`` (int32 [n] on the device), one a row of ``logits`` [n, V]."""
        n, top = tokens.numel(), int(top)
        if n > self.max_batch:
            raise ValueError(f"{n} rows exceed the scorer's batch of {self.max_batch}")
        ring = self._rings.get(top)
        if ring is None:
            ring = self._rings[top] = {"next": 0, "slots": [
                {"host": torch.zeros((3 + 2 * top) * self.max_batch, dtype=torch.float32, pin_memory=True), "event": None} for _ in range(self._depth)]}
        slot = ring["slots"][ring["next"]]
        ring["next"] = (ring["next"] + 1) % self._depth
        if slot["event"] is not None:
            slot["event"].synchronize()
        with torch.cuda.device(self.device):
            # token | log probability | entropy | alternatives' log probabilities | their ids, n (or n * top) numbers each
            out = torch.empty((3 + 2 * top) * n, dtype=torch.float32, device=self.device)
            tokens = tokens.reshape(n, 1)
            out[:n].view(torch.int32).copy_(tokens[:, 0])
            ids = out[(3 + top) * n:].view(torch.int32).view(n, top)
            kernels.token_logprobs(logits, tokens, out[n:2 * n].view(n, 1), out[2 * n:3 * n], out[3 * n:(3 + top) * n].view(n, top), ids)
            slot["host"][:out.numel()].copy_(out, non_blocking=True)
            event = torch.cuda.Event()
            event.record()
            slot["event"] = event
        return PendingScores(n, top, slot["host"], event)

    @staticmethod
    def collect(p: PendingScores) -> List[TokenScore]:
        p.event.synchronize()
        n, k = p.n, p.top
        tokens = p.host[:n].view(torch.int32).tolist()
        logprob, entropy = p.host[n:2 * n].tolist(), p.host[2 * n:3 * n].tolist()
        values = p.host[3 * n:(3 + k) * n].view(n, k).tolist()
        ids = p.host[(3 + k) * n:(3 + 2 * k) * n].view(torch.int32).view(n, k).tolist()
        return [TokenScore(t, lp, h, list(zip(i, v))) for t, lp, h, i, v in zip(tokens, logprob, entropy, ids, values)]


def check_top(top, vocab: int) -> int:
    from ..errors import RocmlError
    most = min(kernels.LOGPROBS_MAX_TOP, vocab)
    if not 0 <= int(top) <= most:
        raise RocmlError(f"{top} alternatives a token: 0 to {most} can be had")
    return int(top)
