"""Verifying drafted tokens through the engine where room is short: memory for graphs, nodes of a step, windows, pieces of which one fails; latents that
serve as keys and values."""
import random

import pytest
import torch

from test_trees_gpu import TOL, folders, path_to, random_tree, rel_err, vocab_of        # noqa: F401 (folders is a fixture)
from tiny_models import _dense, _latent, _layer, prompt, write_pipilix

pytestmark = pytest.mark.gpu


def least_memory(eng, max_tokens, max_slots, monkeypatch):
    """The free memory with which an engine like this is just accepted, found through the refusals."""
    from rocml_b200 import MemoryBudget
    lo, hi = 0, 4 << 30
    while hi - lo > 1:
        mid = (lo + hi) // 2
        monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a, m=mid: (m, 180 << 30))
        try:
            eng._check_budget(max_tokens, max_slots)
            hi = mid
        except MemoryBudget:
            lo = mid
    return hi


def test_graphs_of_trees_take_only_memory_that_is_left(folders, monkeypatch):        # noqa: F811
    """An engine that just fits keeps none; the graphs of short prompts come first, then as many of trees as fit, each with logits for all its nodes.
    The answers are the same bits, and a size is captured only when it has come a few times."""
    from rocml_b200 import Engine, StepEntry, TreeEntry
    from rocml_b200.engine.engine import PROMPT_GRAPHS
    vocab = vocab_of("D")
    eng = Engine.from_folder(folders("D"), dtype="bfloat16", max_tokens=1024, max_slots=4)
    model, tokens = eng.model, eng._prompt_graph_tokens
    least = least_memory(eng, 1024, 4, monkeypatch)
    prompts = PROMPT_GRAPHS * model.workspace_bytes(tokens, 4)
    logits = tokens * vocab * 4
    ids, rng = prompt(8, 50, vocab), random.Random(2)
    trees = [random_tree(rng, n, vocab) for n in (9, 40, 100)]
    answers = []
    for spare in (0, prompts, prompts + logits, prompts + (4 << 30)):
        monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (least + spare, 180 << 30))
        eng = Engine(model, max_tokens=1024, max_slots=4)
        slot = eng.new_sequence()
        eng.step([StepEntry(slot, ids)])
        got = []
        for turn in range(6):
            for t, p in trees:
                got.append(eng.tree_logits([TreeEntry(slot, t, p)]).clone())
            if turn == 0:
                assert not eng._tree_graphs
        assert all(torch.equal(a, b) for a, b in zip(got, got[3:]))
        assert len(eng._tree_graphs) == (3 if spare > prompts + logits else 0), spare
        answers.append(got[:3])
    for a in answers:
        for x, y in zip(a, answers[-1]):
            assert rel_err(x, y) < 2 * TOL["bfloat16"]


def test_verify_in_pieces_is_one_act(folders, monkeypatch):        # noqa: F811
    """If a later piece fails, no sequence has grown, no stream has moved on and no page is lost; the same call then gives what it would have given."""
    from rocml_b200 import Engine, SamplingParams, StepEntry, TreeEntry
    from rocml_b200.sampling import XorShift64Star
    vocab = vocab_of("D")
    rng = random.Random(12)
    ctx = [prompt(70 + n, n, vocab) for n in (130, 20, 64, 100)]
    trees = [random_tree(rng, n, vocab) for n in (200, 190, 180, 250)]
    params = [SamplingParams(), SamplingParams(0.8, 40, seed=3), SamplingParams(0.9, 30, None, seed=9, repeat_penalty=1.3), SamplingParams(1.0, seed=4)]

    def start():
        eng = Engine.from_folder(folders("D"), dtype="float32", max_tokens=64 * 40, max_slots=8)
        slots = [eng.new_sequence() for _ in ctx]
        eng.step([StepEntry(s, c) for s, c in zip(slots, ctx)])
        return eng, slots, [TreeEntry(s, t, p) for s, (t, p) in zip(slots, trees)], [XorShift64Star(5 + i) for i in range(4)]
    eng, slots, entries, streams = start()
    histories = [c + [t[0]] for c, (t, _) in zip(ctx, trees)]
    want = eng.verify(entries, params, streams, histories)
    want_lengths, want_next = [eng.length(s) for s in slots], [s.next_f32() for s in streams]
    eng, slots, entries, streams = start()
    run, calls = eng._tree_steps()._run, []

    def failing(piece):
        calls.append(len(piece))
        if len(calls) > 1:
            raise RuntimeError("the second piece")
        return run(piece)
    free = [g.pool.n_free for g in eng.cache.kv_groups]
    with monkeypatch.context() as m:
        m.setattr(eng._tree_steps(), "_run", failing)
        with pytest.raises(RuntimeError, match="second piece"):
            eng.verify(entries, params, streams, histories)
    assert len(calls) == 2 and [eng.length(s) for s in slots] == [len(c) for c in ctx]
    eng.cache.check_invariants()
    assert [g.pool.n_free for g in eng.cache.kv_groups] == free
    assert eng.verify(entries, params, streams, histories) == want
    assert [eng.length(s) for s in slots] == want_lengths and [s.next_f32() for s in streams] == want_next
    eng.cache.check_invariants()


@pytest.mark.parametrize("name,step_tokens", [("A", 4), ("A", 1), ("B", 20), ("C", 4096), ("E", 7), ("PA", 4096), ("PB", 12), ("PC", 4096)])
def test_drafts_that_an_engine_cannot_take_are_cut(folders, name, step_tokens):        # noqa: F811
    """More guesses than a step holds, deeper ones than a window: the answers are the ordinary ones (32-bit), also where no guess is left."""
    from rocml_b200 import Engine, SamplingParams
    vocab = vocab_of(name)
    eng = Engine.from_folder(folders(name), dtype="float32", max_tokens=64 * 12, max_slots=3, max_step_tokens=step_tokens)
    prompts = [prompt(60 + n, n, vocab) for n in (3, 17, 40)]
    params = SamplingParams(0.8, 40, 0.95, seed=5)
    want = eng.generate(prompts, max_new_tokens=14, sampling=params, stop_tokens=[])
    texts = [p + w.tokens for p, w in zip(prompts, want)]

    def drafter(history):
        text = next(t for t in texts if t[:len(history)] == list(history))
        guesses = (text[len(history):] + [1] * 40)[:40]
        tokens, parents, above = [], [], -1
        for g in guesses:                              # a chain of forty, each with a wrong guess beside it
            tokens += [(g + 1) % vocab, g]
            parents += [above, above]
            above = len(tokens) - 1
        return tokens, parents
    got = eng.generate(prompts, max_new_tokens=14, sampling=params, stop_tokens=[], drafter=drafter)
    assert [(g.tokens, g.finish_reason) for g in got] == [(w.tokens, w.finish_reason) for w in want]
    eng.cache.check_invariants()
    assert eng.cache.slots.n_held == 0


@pytest.mark.parametrize("heads,rank", [(16, 64), (20, 128), (8, 48)])
def test_trees_over_latents_in_bfloat16(tmp_path, heads, rank):
    """Layers whose cached rows are keys and values at once: every node's logits against its path as an ordinary prompt, and greedy verifying against the
    most likely tokens."""
    from rocml_b200 import Engine, SamplingParams, StepEntry, TreeEntry
    config = {"architecture": "Pipilix", "vocab": 333, "width": 128, "embedding": {"scale": 1.0}, "norm": {"eps": 1e-5}, "logit_scale": 1.0,
              "layers": [_layer(_latent(heads, 32, 32, rank, 200, 0.18), _dense(160)), _layer(_latent(heads, 16, 24, rank, 300, 0.25), _dense(96))]}
    write_pipilix(str(tmp_path), config, seed=6)
    eng = Engine.from_folder(str(tmp_path), dtype="bfloat16", max_tokens=1024, max_slots=3)
    rng = random.Random(8)
    ctx = [prompt(n, n, 333) for n in (64, 150)]
    slots = [eng.new_sequence() for _ in ctx]
    eng.step([StepEntry(s, c) for s, c in zip(slots, ctx)])
    trees = [random_tree(rng, n, 333) for n in (12, 5)]
    entries = [TreeEntry(s, t, p) for s, (t, p) in zip(slots, trees)]
    logits, row = eng.tree_logits(entries).clone(), 0
    for c, (tokens, parents) in zip(ctx, trees):
        for i in range(len(tokens)):
            way = [tokens[j] for j in path_to(parents, i)]
            slot = eng.new_sequence()
            want = eng.step([StepEntry(slot, c + way, [len(c) + len(way) - 1])])
            eng.release(slot)
            assert rel_err(logits[row:row + 1], want) < 2 * TOL["bfloat16"], i
            row += 1
    # trees that hold the most likely token behind the root, after a wrong one
    best = [int(logits[0].argmax()), int(logits[12].argmax())]
    entries = [TreeEntry(s, [t[0], (b + 1) % 333, b], [-1, 0, 0]) for s, (t, _), b in zip(slots, trees, best)]
    lone = eng.tree_logits(entries).clone()
    got = eng.verify(entries, [SamplingParams()] * 2)
    for i, (c, (t, _), b, g) in enumerate(zip(ctx, trees, best, got)):
        if int(lone[3 * i].argmax()) != b:             # (a near tie fell differently in the other tree)
            continue
        assert g[0] == b and len(g) == 2 and eng.length(slots[i]) == len(c) + 2
        # the row that was moved is read again: as a prompt
        again = eng.step([StepEntry(slots[i], [g[1]], [0])]).clone()
        slot = eng.new_sequence()
        want = eng.step([StepEntry(slot, c + [t[0], b, g[1]], [len(c) + 2])])
        eng.release(slot)
        assert rel_err(again, want) < 2 * TOL["bfloat16"]


@pytest.mark.parametrize("windows", [(50, 7), (9, 50), (None, 12)])
def test_layers_that_read_anothers_cache_through_another_window(tmp_path, windows):
    """Drafts down to the narrowest window change no answer (32-bit); deeper ones are refused."""
    from rocml_b200 import Engine, RocmlError, StepEntry, TreeEntry
    from tiny_models import _KA_ROT, _kdiff, write_kemizen
    config = {"architecture": "Kemizen", "vocab": 211, "width": 64, "embedding": {"scale": 1.5}, "norm": {"eps": 1e-6},
              "layers": [_kdiff(4, 2, 12, 20, 0.5, 0.3, _KA_ROT, 96, size=windows[0], softcap=3.0),
                         _kdiff(4, 2, 12, 20, 0.7, 0.5, _KA_ROT, 48, size=windows[1], softcap=5.0, kv_from=0)]}
    write_kemizen(str(tmp_path), config, seed=4)
    eng = Engine.from_folder(str(tmp_path), dtype="float32", max_tokens=1024, max_slots=3)
    deepest = min(w for w in windows if w)
    ids, way = prompt(5, 70, 211), prompt(6, deepest, 211)
    slot = eng.new_sequence()
    eng.step([StepEntry(slot, ids)])
    got = eng.tree_logits([TreeEntry(slot, way + [3, 4], list(range(-1, deepest - 1)) + [0, 1])]).clone()
    paths = [way[:i + 1] for i in range(deepest)] + [way[:1] + [3], way[:2] + [4]]
    for g, path in zip(got, paths):
        other = eng.new_sequence()
        want = eng.step([StepEntry(other, ids + path, [70 + len(path) - 1])])
        eng.release(other)
        assert rel_err(g[None], want) < 2 * TOL["float32"]
    with pytest.raises(RocmlError, match="window"):
        eng.tree_logits([TreeEntry(slot, way + [1], list(range(-1, deepest)))])


def test_an_engine_that_verified_is_gone_when_it_is_dropped(folders):        # noqa: F811
    """Its memory with it, without waiting for the collector of cycles (which may come while another engine captures a graph, and graphs that go then spoil
    the capture)."""
    import gc
    import weakref
    from rocml_b200 import Engine, PromptLookup
    vocab = vocab_of("D")
    torch.cuda.synchronize()
    gc.collect()
    gc.disable()
    try:
        before = torch.cuda.memory_allocated()
        for use in ("plain", "trees", "drafts", "scores"):
            eng = Engine.from_folder(folders("D"), dtype="bfloat16", max_tokens=1024, max_slots=4)
            assert torch.cuda.memory_allocated() > before
            if use == "plain":
                eng.generate([prompt(1, 20, vocab)], max_new_tokens=5)
            elif use == "trees":
                from rocml_b200 import TreeEntry
                slot = eng.new_sequence()
                for _ in range(4):
                    eng.tree_logits([TreeEntry(slot, [1, 2, 3], [-1, 0, 0])])
                assert eng._tree_graphs
            elif use == "drafts":
                eng.generate([[1, 2, 3] * 5], max_new_tokens=30, drafter=PromptLookup())
            else:
                eng.score([prompt(1, 20, vocab)], top=2)
            gone = weakref.ref(eng)
            del eng
            assert gone() is None, use
    finally:
        gc.enable()


def test_a_capture_is_not_spoiled_by_graphs_that_go(folders, monkeypatch):        # noqa: F811
    """An engine in a cycle of references, found by the collector while another captures: its graphs go after the capture."""
    import gc
    from rocml_b200 import Engine, StepEntry
    vocab = vocab_of("D")

    def steps(eng):
        slot = eng.new_sequence()
        eng.step([StepEntry(slot, prompt(1, 20, vocab))])
        return torch.cat([eng.step([StepEntry(slot, [t], [0])]).clone() for t in (3, 4, 5)])
    old = Engine.from_folder(folders("D"), dtype="bfloat16", max_tokens=1024, max_slots=4)
    want = steps(old)
    old.itself, held = old, [old]
    del old
    eng = Engine.from_folder(folders("D"), dtype="bfloat16", max_tokens=1024, max_slots=4)
    forward, captured = eng.model.forward, []

    def drops(batch, cache):
        if batch.capturing:
            captured.append(len(held))
            held.clear()
            if gc.isenabled():                         # (the collector's turn, which comes whenever it is allowed to)
                gc.collect()
        return forward(batch, cache)
    monkeypatch.setattr(eng.model, "forward", drops)
    assert torch.equal(steps(eng), want)
    assert captured == [1] and gc.isenabled() and eng.graphs_captured == 1
