"""Limits of drafted tokens and of scoring without a GPU: windows of layers that share a cache, nodes and sequences of a step, guesses that are too many, memory
that scoring holds."""
import contextlib
import random
import weakref
from types import SimpleNamespace

import pytest
import torch

from rocml_b200 import kernels
from rocml_b200.cache import SequenceCache
from rocml_b200.errors import KernelError, RocmlError


class Parts(SimpleNamespace):
    """What of an engine is asked for."""


@pytest.mark.parametrize("keeper,reader,deepest", [(50, 7, 7), (9, 50, 9), (None, 8, 8), (12, None, 12), (None, None, 256)])
def test_the_narrowest_window_of_any_layer_bounds_a_tree(keeper, reader, deepest):
    """Also where the cache keeps more, for another layer that reads it."""
    from rocml_b200.config import config_from_dict
    from rocml_b200.engine.model import Model
    from rocml_b200.engine.trees import TreeEntry, TreeSteps
    from rocml_b200.parts import BuildEnv
    from tiny_models import _KA_ROT, _kdiff
    cfg = {"architecture": "Kemizen", "vocab": 211, "width": 64, "embedding": {"scale": 1.5}, "norm": {"eps": 1e-6},
           "layers": [_kdiff(4, 2, 12, 20, 0.5, 0.3, _KA_ROT, 96, size=keeper), _kdiff(4, 2, 12, 20, 0.7, 0.5, _KA_ROT, 48, size=reader, kv_from=0)]}
    model = Model(config_from_dict(cfg).to_model_spec(), BuildEnv(torch.device("cpu"), torch.float32))
    cache = SequenceCache(model.cache_requirements(), model.reads_cache_of(), 1024, 2, 1024, torch.float32, torch.device("cpu"), 512)
    engine = Parts(model=model, cache=cache, max_step_tokens=512)
    steps = TreeSteps(engine)
    slot = cache.alloc_slot()
    chain = lambda n: TreeEntry(slot, [1] * n, list(range(-1, n - 1)))
    assert steps._check([chain(deepest)])
    assert steps._check([TreeEntry(slot, [1] * 200, [-1] + [0] * 199)])
    if deepest < 256:
        with pytest.raises(RocmlError, match=f"window holds {deepest} positions"):
            steps._check([chain(deepest + 1)])


def test_an_engines_limits_cut_drafts():
    """The loop's decisions with an engine that says what a tree may be: the ordinary answers, never more nodes or deeper ones."""
    from rocml_b200.engine.drafting import generate_drafted
    from rocml_b200.engine.generate import Request, generate
    from rocml_b200.sampling import SamplingParams
    from test_drafting import Fake

    class Limited(Fake):
        def verify(self, entries, params, rngs, histories):
            for e in entries:
                depth = []
                for p in e.parents:
                    depth.append(depth[p] + 1 if p >= 0 else 1)
                assert len(e.tokens) <= self.tree_limits[0] and max(depth) <= self.tree_limits[1]
                self.deepest = max(self.deepest, max(depth))
            return super().verify(entries, params, rngs, histories)

    for limits in ((1, 256), (2, 256), (9, 3), (256, 1), (256, 2), (30, 30)):
        rng = random.Random(sum(limits))
        reqs = [Request([rng.randrange(10) for _ in range(rng.randrange(1, 20))], 25, SamplingParams(), stop_tokens=[]) for _ in range(5)]

        def drafter(history):
            text, tokens, parents, above = list(history), [], [], -1
            for _ in range(40):
                guess = Fake.follow(text)
                for g in ([guess, rng.randrange(11)] if rng.random() < 0.5 else [rng.randrange(11), guess]):
                    tokens.append(g)
                    parents.append(above)
                above = next(i for i in range(len(tokens)) if parents[i] == above and tokens[i] == guess)
                text.append(guess)
            return tokens, parents
        plain, limited = Fake(), Limited()
        limited.tree_limits, limited.deepest = limits, 0
        want, got = generate(plain, reqs, max_batch=3), generate_drafted(limited, reqs, drafter, max_batch=3)
        assert [(c.tokens, c.finish_reason) for c in got] == [(c.tokens, c.finish_reason) for c in want]
        assert max(limited.nodes) <= limits[0] and (limited.steps < plain.steps) == (min(limits) > 1)
        assert limited.deepest == 1 if min(limits) == 1 else limited.deepest > 1
    for parents in ([-1, 1], [-1, 5], [-2, 0]):
        fake = Fake()
        with pytest.raises(RocmlError, match="earlier"):
            generate_drafted(fake, [Request([1, 2, 3], 5)], lambda h: ([1, 2], parents))
        assert not fake.text


def test_a_step_takes_no_more_sequences_than_its_kernels():
    from rocml_b200.engine.trees import TreeEntry, TreeSteps
    steps = TreeSteps.__new__(TreeSteps)
    steps.max_nodes = 4096
    entries = [TreeEntry(i, [1] * (1 + i % 3 // 2), [-1, 0][:1 + i % 3 // 2]) for i in range(2500)]
    pieces = list(steps._pieces(entries))
    assert [e for p in pieces for e in p] == entries and all(0 < len(p) <= kernels.TREE_MAX_SEQS for p in pieces)
    assert all(sum(len(e.tokens) for e in p) <= 4096 for p in pieces) and len(pieces) == 3


@pytest.mark.parametrize("vocab", [300, 151936, 262144, 2 ** 27])
def test_scoring_holds_the_logits_of_one_piece(vocab, monkeypatch):
    """A piece's logits go before the next one's come, and are no more than 320 MiB (one row at least)."""
    from rocml_b200.engine import scoring
    from rocml_b200.sampling import TokenScore
    alive, rows = [], []

    def step(entries):
        assert not any(r() is not None for r in alive)
        n = len(entries[0].tokens)
        rows.append(n)
        logits = torch.zeros((n, 1))
        alive.append(weakref.ref(logits))
        return logits

    class Scorer:
        def __init__(self, device, max_batch, depth):
            self.max_batch = max_batch

        def launch(self, logits, tokens, top):
            assert logits.shape[0] == tokens.numel() <= self.max_batch
            return tokens.tolist()

        @staticmethod
        def collect(tokens):
            return [TokenScore(t, 0.0, 0.0, []) for t in tokens]
    monkeypatch.setattr(scoring, "Scorer", Scorer)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(kernels, "check_status", lambda d: None)
    engine = SimpleNamespace(model=SimpleNamespace(vocab=vocab), max_seq_len=4000, max_step_tokens=4096, device=torch.device("cpu"), step=step,
                             new_sequence=lambda: 0, release=lambda s: None)
    text = [i % 299 for i in range(1100 if vocab < 2 ** 27 else 5)]
    got = scoring.score(engine, [text, text[:2]])
    assert [[s.token for s in g] for g in got] == [text[1:], text[1:2]]
    assert max(rows) == max(1, min(512, (320 << 20) // (4 * vocab)))


class _OnAnotherDevice(torch.Tensor):
    def get_device(self):
        return 5


def test_a_sink_on_another_device_is_refused():
    from test_tree import _attention
    with pytest.raises(KernelError, match="one device"):
        _attention(sink=torch.zeros(8).as_subclass(_OnAnotherDevice))


@pytest.mark.parametrize("hd", [16, 64, 80, 128, 256, 512])
@pytest.mark.parametrize("group,nkv", [(1, 1), (4, 8), (7, 3), (128, 1), (2, 400)])
def test_no_call_works_in_more_than_the_budget_counts(hd, group, nkv, monkeypatch):
    monkeypatch.setattr(kernels, "_decode_slots", lambda device: 444)
    most = kernels.tree_work_bytes(nkv, hd, 0)
    for tensor_cores in {False, hd in (64, 128, 256)}:
        for n_seqs in (1, 2, 5, 16, 33, 37, 256):
            for nodes in (1, 9, 33, 256):
                for pages in (1, 2, 7, 16, 64, 3000):
                    plan = kernels._tree_plan.__wrapped__(tensor_cores, n_seqs, nodes, group, nkv, hd, pages, 0)
                    assert 4 * plan[3] <= most
