"""Drafted tokens without a GPU: trees as a step packs them, pages given back, the loop's decisions, drafts from the text, scores asked for."""
import random

import numpy as np
import pytest
import torch

from rocml_b200.cache import SequenceCache
from rocml_b200.cache.requirements import KVRequirement
from rocml_b200.engine.drafting import PromptLookup, generate_drafted
from rocml_b200.engine.generate import GenerateStats, Request, generate
from rocml_b200.engine.trees import TreeEntry, check_tree, pack_trees
from rocml_b200.errors import RocmlError
from rocml_b200.sampling import SamplingParams, TokenScore


def test_pack_trees():
    positions, parents, bits, depths = pack_trees([10, 0], [[-1, 0, 0, 2, 1], [-1] + list(range(255))])
    assert positions[:5] == [10, 11, 11, 12, 12] and depths[:5] == [0, 1, 1, 2, 2] and parents[:5] == [-1, 0, 0, 2, 1]
    assert [int(b) for b in bits[:5, 0]] == [0b1, 0b11, 0b101, 0b1101, 0b10011] and (bits[:5, 1:] == 0).all()
    assert positions[5:] == list(range(256)) and bits.shape == (261, 8) and bits.dtype == np.int32
    assert (bits[-1] == -1).all() and bits[5 + 31].tolist() == [-1] + [0] * 7


@pytest.mark.parametrize("tokens,parents", [([], []), ([1, 2], [-1]), ([1, 2], [-1, -1]), ([1, 2], [0, 0]), ([1, 2, 3], [-1, 2, 0]),
                                            ([1, 99], [-1, 0]), ([1] * 257, [-1] + [0] * 256)])
def test_check_tree_refuses(tokens, parents):
    with pytest.raises(RocmlError):
        check_tree(TreeEntry(0, tokens, parents), vocab=50)


def test_pages_of_tokens_that_were_not_kept_come_back():
    for window in (None, 100):
        c = SequenceCache([KVRequirement(1, 16, window), KVRequirement(2, 16)], [None, None], 1024, 4, 1024, torch.float32, torch.device("cpu"), 64)
        a, b = c.alloc_slot(), c.alloc_slot()
        c.grow(a, 300)
        c.commit(a, 300)
        c.grow(b, 64)
        c.commit(b, 64)
        free = [g.pool.n_free for g in c.kv_groups]
        c.grow(a, 200)                       # a tree of 200 nodes, of which 3 are kept
        c.commit(a, 3)
        c.trim(a)
        c.check_invariants()
        assert c.length(a) == 303 and [g.pool.n_free for g in c.kv_groups] == free
        c.grow(a, 18)                        # into another page
        c.commit(a, 18)
        c.trim(a)
        c.trim(b)
        c.check_invariants()
        assert c.kv_groups[1].pool.n_free == free[1] - 1
        c.free_slot(a)
        c.free_slot(b)
        c.check_invariants()


def test_prompt_lookup():
    d = PromptLookup(longest=2, length=3, branches=2)
    # "5 6" stood twice before; the later place first, common beginnings shared
    tokens, parents = d([5, 6, 7, 8, 9, 5, 6, 7, 1, 2, 5, 6])
    assert tokens == [7, 1, 2, 8, 9] and parents == [-1, 0, 1, 0, 3]
    # nothing for two tokens: one
    assert d([6, 3, 9, 6]) == ([3, 9, 6], [-1, 0, 1])
    assert d([1, 2, 3]) == ([], []) and d([4]) == ([], [])
    with pytest.raises(RocmlError):
        PromptLookup(length=200, branches=2)


class Fake:
    """An engine whose model continues every sequence by a rule: token t is followed by (3 t + length) % 11, and 10 now and then."""

    def __init__(self, tokens=4096, slots=3, limit=200):
        self.max_seq_len, self._tokens, self._slots = limit, tokens, slots
        self.text, self.released, self.steps, self.nodes = {}, [], 0, []

    def capacity_tokens(self):
        return self._tokens

    def capacity_slots(self):
        return self._slots

    def new_sequence(self):
        s = next(i for i in range(self._slots) if i not in self.text)
        self.text[s] = []
        return s

    def release(self, slot):
        del self.text[slot]
        self.released.append(slot)

    @staticmethod
    def follow(text):
        return (3 * text[-1] + len(text)) % 11

    def run(self, slots, tokens, params, rngs, histories):
        self.steps += 1
        out = []
        for s, t in zip(slots, tokens):
            self.text[s] += t
            assert len(self.text[s]) <= self.max_seq_len
            out.append(self.follow(self.text[s]))
        return out

    def verify(self, entries, params, rngs, histories):
        self.steps += 1
        out = []
        for e, h in zip(entries, histories):
            check_tree(e, 11)
            assert self.text[e.slot] == list(h)[:-1] and e.tokens[0] == h[-1]
            assert len(self.text[e.slot]) + len(e.tokens) <= self.max_seq_len
            self.nodes.append(len(e.tokens))
            self.text[e.slot].append(e.tokens[0])
            here, got = 0, []
            while True:
                t = self.follow(self.text[e.slot])
                got.append(t)
                nxt = next((i for i, (u, p) in enumerate(zip(e.tokens, e.parents)) if p == here and u == t), None)
                if nxt is None:
                    break
                here = nxt
                self.text[e.slot].append(t)
            out.append(got)
        return out


@pytest.mark.parametrize("seed", range(25))
def test_drafted_answers_are_the_ordinary_ones(seed):
    """Right and wrong guesses, stop tokens in the middle of a path, budgets and contexts that end inside one."""
    rng = random.Random(seed)
    reqs = [Request([rng.randrange(10) for _ in range(rng.randrange(1, 20))], rng.choice([0, 1, 2, 5, 40]), SamplingParams(),
                    stop_tokens=[] if rng.random() < 0.5 else [rng.randrange(11)]) for _ in range(7)]

    def drafter(history):
        text, tokens, parents, above = list(history), [], [], -1
        for _ in range(rng.randrange(0, 9)):
            guess = Fake.follow(text) if rng.random() < 0.8 else rng.randrange(11)
            if rng.random() < 0.3:
                tokens.append(rng.randrange(11))
                parents.append(above)
            tokens.append(guess)
            parents.append(above)
            above = len(tokens) - 1
            text.append(guess)
        return tokens, parents

    plain, drafted = Fake(limit=40), Fake(limit=40)
    want = generate(plain, reqs, max_batch=3)
    stats, seen = GenerateStats(), []
    got = generate_drafted(drafted, reqs, drafter, max_batch=3, stats=stats, on_token=lambda i, t: seen.append((i, t)))
    assert [(c.tokens, c.finish_reason) for c in got] == [(c.tokens, c.finish_reason) for c in want]
    assert sorted(i for i, _ in seen) == sorted(i for i, c in enumerate(got) for _ in c.tokens)
    assert not drafted.text and drafted.steps <= plain.steps
    assert stats.prompt_tokens == sum(len(r.prompt) for r in reqs if r.max_new_tokens > 0)


def test_drafted_generation_refuses():
    with pytest.raises(RocmlError, match="empty prompt"):
        generate_drafted(Fake(), [Request([])], PromptLookup())
    with pytest.raises(RocmlError, match="do not come with drafts"):
        generate_drafted(Fake(), [Request([1], logprobs=2)], PromptLookup())
    fake = Fake()
    with pytest.raises(RocmlError, match="3 tokens and 2 parents"):
        generate_drafted(fake, [Request([1, 2, 3], 5), Request([4], 1), Request([5], 5)], lambda h: ([1, 2, 3], [-1, 0]))
    assert not fake.text                      # every slot is back


class Scoring(Fake):
    def launch(self, slots, tokens, params, rngs, histories, feed_from=None, logprobs=None):
        if feed_from is not None:
            tokens = [[t] for t in feed_from["tokens"]]
        out = self.run(slots, tokens, params, rngs, histories)
        return {"tokens": out, "scores": None if logprobs is None else [TokenScore(t, -0.5 * t, 1.0, [(t, -0.1)] * logprobs) for t in out]}

    def collect(self, handle):
        return handle["tokens"]

    def collect_scores(self, handle):
        return handle["scores"]


def test_scores_come_with_the_tokens_that_asked():
    reqs = [Request([1, 2], 6, stop_tokens=[], logprobs=3), Request([3], 4, stop_tokens=[]), Request([4, 4], 5, stop_tokens=[], logprobs=0)]
    want = generate(Fake(), reqs[1:2])
    for ahead in (True, False):
        got = generate(Scoring(), reqs, max_batch=3, run_ahead=ahead)
        assert [len(c.tokens) for c in got] == [6, 4, 5] and got[1].tokens == want[0].tokens
        assert [s.token for s in got[0].logprobs] == got[0].tokens and all(len(s.top) == 3 for s in got[0].logprobs)
        assert got[1].logprobs is None and all(s.top == [] for s in got[2].logprobs) and len(got[2].logprobs) == 5
    with pytest.raises(RocmlError, match="does not score"):
        generate(Fake(), reqs)
