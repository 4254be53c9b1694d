"""How likely given tokens are: prompts run as any prompt does, their logits scored on the GPU."""
from __future__ import annotations

from typing import List, Sequence

import torch

from ..errors import RocmlError
from ..sampling.scorer import Scorer, TokenScore, check_top

# Rows of logits that are scored at a time, and their bytes at most: less than half of the head room of the engine's memory budget (512 rows are 297 MiB at a
# vocabulary of 151,936; a vocabulary of 262,144 takes 320 rows).  One piece's are held at a time.
SCORE_ROWS = 512
SCORE_BYTES = 320 << 20


def score(engine, sequences: Sequence[Sequence[int]], top: int = 0) -> List[List[TokenScore]]:
    """See ``Engine.score``.  Sequence after sequence, in pieces of ``SCORE_ROWS`` tokens at most; each takes a slot and gives it back."""
    from .engine import StepEntry
    top = check_top(top, engine.model.vocab)
    sequences = [[int(t) for t in s] for s in sequences]
    for i, s in enumerate(sequences):
        if not s:
            raise RocmlError(f"sequence {i} is empty")
        if len(s) - 1 > engine.max_seq_len:
            raise RocmlError(f"sequence {i}: {len(s)} tokens exceed the context of {engine.max_seq_len}")
        bad = [t for t in s if not 0 <= t < engine.model.vocab]
        if bad:
            raise RocmlError(f"sequence {i}: token id {bad[0]} is outside the vocabulary of {engine.model.vocab}")
    rows = min(SCORE_ROWS, max(1, SCORE_BYTES // (4 * engine.model.vocab)), engine.max_step_tokens)
    scorer = Scorer(engine.device, max_batch=rows, depth=2)
    out = []
    for s in sequences:
        found: List[TokenScore] = []
        slot = engine.new_sequence()
        try:
            waiting = None
            for a in range(0, len(s) - 1, rows):
                piece = s[a:min(a + rows, len(s) - 1)]
                logits = engine.step([StepEntry(slot, piece, range(len(piece)))])
                with torch.cuda.device(engine.device):
                    after = torch.tensor(s[a + 1:a + 1 + len(piece)], dtype=torch.int32).to(engine.device)
                    pending = scorer.launch(logits, after, top)
                del logits                       # (before the next piece's are made; the memory is used again in the stream's order)
                if waiting is not None:
                    found += scorer.collect(waiting)
                waiting = pending
            if waiting is not None:
                found += scorer.collect(waiting)
        finally:
            engine.release(slot)
        from .. import kernels
        kernels.check_status(engine.device)
        out.append(found)
    return out
