"""Generation that verifies drafted tokens several at a time.

A *drafter* is called with a sequence's tokens so far (prompt and answer) and returns (tokens, parents): guesses at what follows,
``parents[i]`` the earlier guess that guess i follows, -1 where it follows the sequence's last token.  Guesses cost a step's extra rows; those that the
model would have sampled itself save a step each.  The answers are those of ordinary generation with the same parameters, but for near ties:
verifying rounds otherwise than a step of single tokens (other kernels, other orders of sums), so where two tokens are equally likely within rounding, or a draw falls
that close to a border, the other one may come.  In bfloat16 that happens; in 32 bits hardly ever.

What a draft has to bring.  A verifying step costs more than a decode step (contexts of 1,000 tokens, trees of 8 nodes: 1.3 times at 8b sizes and 1.8 at 0.6b, eight
sequences 1.4 and 2.0), also where there is no guess, and the drafter's time on the host comes on top: ``PromptLookup`` looks through the whole text, 0.3 ms a
sequence at 1,000 tokens without a match, 8 ms at 30,000.
"""
from __future__ import annotations

import time
from typing import Callable, Iterable, List, Optional, Sequence, Tuple

from ..errors import RocmlError
from ..sampling.params import XorShift64Star
from .generate import Completion, GenerateStats, Request, decide, plan_batches
from .trees import MAX_NODES, TreeEntry

Drafter = Callable[[Sequence[int]], Tuple[Sequence[int], Sequence[int]]]


class PromptLookup:
    """Drafts from the text itself: where the last tokens (``longest`` of them, else fewer, down to one) stood before, what followed them is the
    guess.  Up to ``branches`` earlier places, the latest first, of ``length`` tokens each, share their common beginnings."""

    def __init__(self, longest: int = 3, length: int = 8, branches: int = 2):
        if longest < 1 or length < 1 or branches < 1 or length * branches >= MAX_NODES:
            raise RocmlError(f"PromptLookup: at least one of each, and fewer than {MAX_NODES} nodes")
        self.longest, self.length, self.branches = longest, length, branches

    def __call__(self, history: Sequence[int]) -> Tuple[List[int], List[int]]:
        history = list(history)
        tokens: List[int] = []
        parents: List[int] = []
        for n in range(min(self.longest, len(history) - 1), 0, -1):
            tail, found = history[-n:], 0
            for at in range(len(history) - n - 1, -1, -1):
                if history[at:at + n] != tail:
                    continue
                above = -1
                for t in history[at + n:at + n + self.length]:
                    same = [i for i, (u, p) in enumerate(zip(tokens, parents)) if p == above and u == t]
                    if same:
                        above = same[0]
                    else:
                        tokens.append(t)
                        parents.append(above)
                        above = len(tokens) - 1
                found += 1
                if found >= self.branches:
                    break
            if found:
                break
        return tokens, parents


def _cut(tokens, parents, most: int, deepest: int) -> Tuple[List[int], List[int]]:
    """The first ``most`` of the guesses that lie no deeper than ``deepest`` below the sequence's last token, parents renumbered."""
    kept, ups, place, depth = [], [], {-1: -1}, {-1: 0}
    for i, (token, up) in enumerate(zip(tokens, parents)):
        if len(kept) >= most:
            break
        if not -1 <= up < i:
            raise RocmlError(f"the drafter's guess {i} follows guess {up}: it must be -1 or an earlier one")
        depth[i] = depth[up] + 1
        if depth[i] <= deepest:
            place[i] = len(kept)
            kept.append(token)
            ups.append(place[up])
    return kept, ups


def _entry(slot: int, history: Sequence[int], drafter: Drafter, room: int, nodes: int, depth: int) -> TreeEntry:
    """The sequence's last token and the drafter's guesses below it, as many as there is room for and as a tree may have, ``nodes`` of them and
    ``depth`` on a path (their parents come first, so what a guess follows is kept with it)."""
    tokens, parents = drafter(history)
    if len(tokens) != len(parents):
        raise RocmlError(f"the drafter gave {len(tokens)} tokens and {len(parents)} parents")
    tokens, parents = _cut(tokens, [int(p) for p in parents], min(room, nodes) - 1, depth - 1)
    return TreeEntry(slot, [history[-1]] + tokens, [-1] + [p + 1 for p in parents])


def generate_drafted(engine, requests: Sequence[Request], drafter: Drafter, default_stop: Iterable[int] = (), max_batch: int = 64,
                     on_token: Optional[Callable[[int, int], bool]] = None, stats: Optional[GenerateStats] = None) -> List[Completion]:
    """``generate`` with drafts: the same requests, and the same answers but for near ties (see above)."""
    stats = stats if stats is not None else GenerateStats()
    default_stop = set(default_stop)
    limit = engine.max_seq_len
    needs = []
    for i, r in enumerate(requests):
        if len(r.prompt) == 0:
            raise RocmlError(f"request {i} has an empty prompt")
        if len(r.prompt) > limit:
            raise RocmlError(f"request {i}: prompt of {len(r.prompt)} tokens exceeds the context of {limit}")
        if r.logprobs is not None:
            raise RocmlError(f"request {i}: log probabilities do not come with drafts (Engine.score gives them afterwards)")
        needs.append(min(len(r.prompt) + max(r.max_new_tokens, 0), limit))
    results: List[Optional[Completion]] = [None] * len(requests)
    for batch in plan_batches(needs, max_batch, engine.capacity_tokens(), engine.capacity_slots()):
        stats.batches += 1
        live = []
        for j, i in enumerate(batch):
            r = requests[i]
            if r.max_new_tokens <= 0:
                results[i] = Completion([], "length", len(r.prompt))
                continue
            live.append({"i": i, "req": r, "slot": engine.new_sequence(), "out": [], "history": list(r.prompt), "need": needs[i],
                         "stops": default_stop if r.stop_tokens is None else set(r.stop_tokens), "rng": XorShift64Star(r.sampling.seed + j)})

        def entry(s) -> TreeEntry:
            nodes, depth = getattr(engine, "tree_limits", (MAX_NODES, MAX_NODES))
            return _entry(s["slot"], s["history"], drafter, s["need"] - len(s["history"]) + 1, nodes, depth)

        def take(s, tokens) -> bool:
            """Append what was sampled; whether the sequence goes on."""
            r = s["req"]
            for tok in tokens:
                emit, reason = decide(tok, len(s["out"]), r.max_new_tokens, len(s["history"]) + 1, limit, s["stops"], r.ignore_eos)
                if emit:
                    s["out"].append(tok)
                    s["history"].append(tok)
                    if on_token is not None and on_token(s["i"], tok) and reason is None:
                        reason = "stop"
                if reason is not None:
                    engine.release(s["slot"])
                    results[s["i"]] = Completion(s["out"], reason, len(r.prompt))
                    return False
            return True

        try:
            _run_batch(engine, live, entry, take, stats)
        except BaseException:
            for s in live:                    # (a drafter may fail: the sequences that were running give their slots back)
                if results[s["i"]] is None:
                    engine.release(s["slot"])
            raise
    return results


def _run_batch(engine, live, entry, take, stats) -> None:
    """Prompts, then drafts (``entry`` of a sequence) until every sequence has ended."""
    first = True
    while live:
        t0 = time.perf_counter()
        before = sum(len(s["out"]) for s in live)
        if first:
            sampled = [[t] for t in engine.run([s["slot"] for s in live], [s["history"] for s in live], [s["req"].sampling for s in live],
                                               [s["rng"] for s in live], [s["history"] for s in live])]
        else:
            sampled = engine.verify([entry(s) for s in live], [s["req"].sampling for s in live], [s["rng"] for s in live], [s["history"] for s in live])
        running = live
        live = [s for s, tokens in zip(running, sampled) if take(s, tokens)]
        dt = time.perf_counter() - t0
        stats.step_batch_sizes.append(len(running))
        if first:
            stats.prefill_seconds += dt
            stats.prompt_tokens += sum(len(s["req"].prompt) for s in running)
            first = False
        else:
            stats.decode_seconds += dt
            stats.decode_tokens += sum(len(s["out"]) for s in running) - before
