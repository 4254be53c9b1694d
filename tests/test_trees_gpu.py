"""Trees of drafted tokens through the engine, against the same tokens taken in ordinary steps; generation with drafts; scoring."""
import random

import pytest
import torch

from tiny_models import CONFIGS, PIPILIX, SAFESUN, prompt, write_model, write_pipilix, write_safesun

pytestmark = pytest.mark.gpu

TOL = {"float32": 2e-5, "bfloat16": 2.5e-2}      # tests/test_engine_gpu.py says what of; two engine results differ by twice that at most


def rel_err(got, want):
    scale = want.double().abs().amax(dim=-1, keepdim=True).clamp_min(1e-30)
    return float(((got.double() - want.double()).abs() / scale).max())


def vocab_of(name):
    return {**CONFIGS, **PIPILIX, **SAFESUN}[name].get("vocab_size") or {**PIPILIX, **SAFESUN}[name]["vocab"]


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    made = {}

    def get(name):
        if name not in made:
            folder = str(tmp_path_factory.mktemp(f"tree_{name}"))
            if name in CONFIGS:
                write_model(folder, CONFIGS[name], seed=31, std=0.06)
            elif name in PIPILIX:
                write_pipilix(folder, PIPILIX[name], seed=32)
            else:
                write_safesun(folder, SAFESUN[name], seed=33)
            made[name] = folder
        return made[name]
    return get


def random_tree(rng, n, vocab):
    return [rng.randrange(vocab) for _ in range(n)], [-1] + [rng.randrange(max(0, i - 4), i) for i in range(1, n)]


def path_to(parents, i):
    way = []
    while i >= 0:
        way.append(i)
        i = parents[i]
    return way[::-1]


@pytest.mark.parametrize("name,dtype", [(n, d) for n in ("A", "B", "C", "D", "E", "SA", "SB") for d in ("float32", "bfloat16")] + [("PA", "float32"), ("PB", "float32")])
def test_tree_logits_are_those_of_the_paths(folders, name, dtype):
    """Every node's logits against the last logits of context and path taken as an ordinary prompt; twice, a tree leaving nothing behind."""
    from rocml_b200 import Engine, StepEntry, TreeEntry
    vocab = vocab_of(name)
    eng = Engine.from_folder(folders(name), dtype=dtype, max_tokens=2048, max_slots=8)
    if not eng.model.takes_trees:
        pytest.skip("a model without trees")
    rng = random.Random(7)
    contexts = [c for c in (5, 63, 64, 90) if c + 12 <= eng.max_seq_len]
    ctx = [prompt(40 + c, c, vocab) for c in contexts]
    trees = [random_tree(rng, n, vocab) for n in (9, 1, 6, 4)[:len(ctx)]]
    windows = [g.req.window for g in eng.cache.kv_groups if g.req.window]
    deepest = max(len(path_to(p, i)) for _, p in trees for i in range(len(p)))
    slots = [eng.new_sequence() for _ in ctx]
    eng.step([StepEntry(s, c) for s, c in zip(slots, ctx)])
    entries = [TreeEntry(s, t, p) for s, (t, p) in zip(slots, trees)]
    if windows and deepest > min(windows):
        from rocml_b200 import RocmlError
        with pytest.raises(RocmlError, match="window"):
            eng.tree_logits(entries)
        return
    got = [eng.tree_logits(entries).clone() for _ in range(2)]
    assert [eng.length(s) for s in slots] == contexts
    eng.cache.check_invariants()
    # (the sequences carry on as if nothing had been)
    after = eng.step([StepEntry(s, [t[0]], [0]) for s, (t, _) in zip(slots, trees)]).clone()
    row = 0
    for b, (c, (tokens, parents)) in enumerate(zip(ctx, trees)):
        for i in range(len(tokens)):
            way = [tokens[j] for j in path_to(parents, i)]
            slot = eng.new_sequence()
            want = eng.step([StepEntry(slot, c + way, [len(c) + len(way) - 1])])
            eng.release(slot)
            for g in got:
                assert rel_err(g[row:row + 1], want) < 2 * TOL[dtype], (name, b, i)
            if i == 0:
                assert rel_err(after[b:b + 1], want) < 2 * TOL[dtype]
            row += 1


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E", "SA"])
@pytest.mark.parametrize("sampling", ["greedy", "drawn", "penalty"])
def test_drafts_change_no_answer(folders, name, sampling):
    """32-bit: a drafter that knows the ordinary answers and mixes wrong guesses in gives the same tokens in fewer steps, greedy, drawn
    and with a repeat penalty; so does one that looks in the text."""
    from rocml_b200 import Engine, PromptLookup, SamplingParams
    from rocml_b200.engine.generate import GenerateStats
    vocab = vocab_of(name)
    eng = Engine.from_folder(folders(name), dtype="float32", max_tokens=64 * 24, max_slots=4)
    if not eng.model.takes_trees:
        pytest.skip("a model without trees")
    params = {"greedy": SamplingParams(), "drawn": SamplingParams(0.8, 40, 0.95, seed=5),
              "penalty": SamplingParams(0.9, 30, None, seed=9, repeat_penalty=1.3)}[sampling]
    prompts = [prompt(60 + n, n, vocab) for n in (3, 17, 60, 64, 30)]
    plain_stats, stats = GenerateStats(), GenerateStats()
    want = eng.generate(prompts, max_new_tokens=20, sampling=params, stop_tokens=[], max_batch=3, stats=plain_stats)
    texts = [p + w.tokens for p, w in zip(prompts, want)]
    rng = random.Random(3)

    def knows(history):
        text = next(t for t in texts if t[:len(history)] == list(history))
        tokens, parents, above = [], [], -1
        for t in text[len(history):len(history) + 5]:
            wrong = (t + 1 + rng.randrange(vocab - 1)) % vocab
            for u in ([t, wrong] if rng.random() < 0.5 else [wrong, t]):
                tokens.append(u)
                parents.append(above)
            above = len(tokens) - (2 if tokens[-2] == t else 1)
        return tokens, parents

    got = eng.generate(prompts, max_new_tokens=20, sampling=params, stop_tokens=[], max_batch=3, drafter=knows, stats=stats)
    assert [(g.tokens, g.finish_reason) for g in got] == [(w.tokens, w.finish_reason) for w in want]
    assert len(stats.step_batch_sizes) < len(plain_stats.step_batch_sizes) / 2
    got = eng.generate(prompts, max_new_tokens=20, sampling=params, stop_tokens=[], max_batch=3, drafter=PromptLookup())
    assert [g.tokens for g in got] == [w.tokens for w in want]
    eng.cache.check_invariants()
    assert eng.cache.slots.n_held == 0


def test_verify_in_graphs_and_in_pieces(folders):
    """bfloat16, sizes that come back: launched, then replayed from a graph, the same logits and the same path; more nodes than a step holds are taken in
    pieces; room that is not there is refused before anything runs."""
    from rocml_b200 import CacheFull, Engine, SamplingParams, StepEntry, TreeEntry
    vocab = vocab_of("D")
    eng = Engine.from_folder(folders("D"), dtype="bfloat16", max_tokens=64 * 40, max_slots=8)
    assert eng._prompt_graph_tokens > 0
    rng = random.Random(11)
    ctx = [prompt(70 + n, n, vocab) for n in (130, 20, 64)]
    slots = [eng.new_sequence() for _ in ctx]
    eng.step([StepEntry(s, c) for s, c in zip(slots, ctx)])
    trees = [random_tree(rng, n, vocab) for n in (20, 7, 13)]
    entries = [TreeEntry(s, t, p) for s, (t, p) in zip(slots, trees)]
    runs = [eng.tree_logits(entries).clone() for _ in range(3)]
    assert len(eng._tree_graphs) == 1 and eng._replayed
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[1], runs[2])
    # greedy: what is confirmed is the chain of each node's most likely token
    best, row, want = runs[0].argmax(-1).tolist(), 0, []
    for tokens, parents in trees:
        here, got = 0, []
        while here is not None:
            got.append(best[row + here])
            here = next((i for i, p in enumerate(parents) if p == here and tokens[i] == got[-1]), None)
        want.append(got)
        row += len(tokens)
    assert eng.verify(entries, [SamplingParams()] * 3) == want
    assert [eng.length(s) for s in slots] == [len(c) + len(w) for c, w in zip(ctx, want)]
    eng.cache.check_invariants()
    # pieces
    big = [random_tree(rng, 200, vocab) for _ in slots]
    many = [TreeEntry(s, t, p) for s, (t, p) in zip(slots, big)]
    whole = eng.tree_logits(many)
    alone = [eng.tree_logits([e]).clone() for e in many]
    assert whole.shape[0] == 600 and rel_err(whole, torch.cat(alone)) < 2 * TOL["bfloat16"]
    with pytest.raises(CacheFull):
        small = Engine.from_folder(folders("D"), dtype="bfloat16", max_tokens=128, max_slots=2)
        s = [small.new_sequence() for _ in range(2)]
        small.step([StepEntry(x, ctx[1]) for x in s])
        small.verify([TreeEntry(x, *random_tree(rng, 60, vocab)) for x in s], [SamplingParams()] * 2)
    small.cache.check_invariants()
    assert [small.length(x) for x in s] == [20, 20]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_trees_behind_nothing_and_up_to_the_last_place(folders, dtype):
    """A sequence without a context, ordinary steps between verified ones, a tree whose nodes end at the context's last place; one more is refused."""
    from rocml_b200 import ContextOverflow, Engine, SamplingParams, StepEntry, TreeEntry
    vocab = vocab_of("D")
    eng = Engine.from_folder(folders("D"), dtype=dtype, max_tokens=192, max_slots=2, max_seq_len=128)
    greedy = [SamplingParams()]
    ids = prompt(3, 4, vocab)
    slot, other = eng.new_sequence(), eng.new_sequence()
    tree = TreeEntry(slot, [ids[0], ids[1], ids[2], ids[1]], [-1, 0, 1, 0])
    lone = eng.step([StepEntry(other, ids[:3], [0, 1, 2])])
    got = eng.tree_logits([tree])
    assert rel_err(got[:3], lone) < 2 * TOL[dtype] and rel_err(got[3:], lone[1:2]) < 2 * TOL[dtype]
    text = [ids[0]]
    while len(text) < 120:
        # the token that an ordinary step would draw next is among the guesses every third time
        old = eng.length(slot)
        assert old == len(text) - 1
        want = int(eng.tree_logits([TreeEntry(slot, [text[-1]], [-1])]).argmax())
        guess = want if len(text) % 3 == 0 else (want + 1) % vocab
        new = eng.verify([TreeEntry(slot, [text[-1], (want + 2) % vocab, guess], [-1, 0, 0])], greedy)[0]
        assert new[0] == want and len(new) == (2 if guess == want else 1)
        text += new
        if len(text) % 5 == 0:
            logits = eng.step([StepEntry(slot, [text[-1]], [0])])
            text.append(int(logits.argmax()))
    eng.release(other)
    old = eng.length(slot)
    n = 128 - old
    fits = TreeEntry(slot, [text[-1]] + [1] * (n - 1), [-1] + [0] * (n - 1))
    assert eng.tree_logits([fits]).shape[0] == n
    with pytest.raises(ContextOverflow):
        eng.verify([TreeEntry(slot, fits.tokens + [1], fits.parents + [0])], greedy)
    assert eng.length(slot) == old
    eng.cache.check_invariants()


def test_models_that_keep_more_than_keys_and_values_refuse_trees(tmp_path):
    from rocml_b200 import ConfigError, Engine, TreeEntry
    from tiny_models import TIBENEX, write_tibenex
    write_tibenex(str(tmp_path), TIBENEX["TA"], seed=5)
    eng = Engine.from_folder(str(tmp_path), dtype="float32", max_tokens=256)
    with pytest.raises(ConfigError, match="trees"):
        eng.tree_logits([TreeEntry(eng.new_sequence(), [1], [-1])])


# ---- scoring ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_scores_are_the_plain_implementations(folders, name):
    """float32 engine logits are within 2e-5 of the row's largest logit of the plain ones (tests/test_engine_gpu.py), and a log probability moves by
    at most twice what its logits do."""
    from plain_qwen3 import PlainQwen3
    from rocml_b200 import Engine
    plain = PlainQwen3(folders(name), dtype=torch.float64)
    vocab = vocab_of(name)
    eng = Engine.from_folder(folders(name), dtype="float32", max_tokens=1024, max_slots=4, max_step_tokens=50)
    texts = [prompt(80 + n, n, vocab) for n in (1, 2, 40, 120)]
    for text, got in zip(texts, eng.score(texts, top=4)):
        assert [s.token for s in got] == text[1:]
        if len(text) == 1:
            continue
        logits = plain.logits(text)[:-1].double()
        logp = torch.log_softmax(logits, -1)
        tol = 4e-5 * float(logits.abs().max()) + 1e-5
        for i, s in enumerate(got):
            assert abs(s.logprob - float(logp[i, text[i + 1]])) < tol
            assert abs(s.entropy + float((logp[i].exp() * logp[i]).sum())) < tol * 10
            values = sorted(logp[i].tolist(), reverse=True)[:4]
            assert all(abs(v - w) < tol for (_, v), w in zip(s.top, values)) and all(abs(float(logp[i, t]) - v) < tol for t, v in s.top)
    assert eng.cache.slots.n_held == 0


def test_generated_tokens_come_with_their_scores(folders):
    """Each token's score is what scoring the finished text says of it, with and without running ahead; most likely first under greedy."""
    from rocml_b200 import Engine, RocmlError, SamplingParams
    vocab = vocab_of("B")
    eng = Engine.from_folder(folders("B"), dtype="float32", max_tokens=1024, max_slots=4)
    prompts = [prompt(90 + n, n, vocab) for n in (4, 33, 12)]
    plain = eng.generate(prompts, max_new_tokens=9, stop_tokens=[], max_batch=2)
    for ahead in (True, False):
        outs = eng.generate(prompts, max_new_tokens=9, stop_tokens=[], max_batch=2, logprobs=3, run_ahead=ahead)
        assert [o.tokens for o in outs] == [o.tokens for o in plain]
        for p, o in zip(prompts, outs):
            told = eng.score([p + o.tokens], top=3)[0][len(p) - 1:]
            assert [s.token for s in o.logprobs] == o.tokens
            for a, b in zip(o.logprobs, told):
                assert abs(a.logprob - b.logprob) < 1e-4 and a.top[0][0] == a.token and [t for t, _ in a.top] == [t for t, _ in b.top]
    drawn = eng.generate(prompts, max_new_tokens=9, sampling=SamplingParams(0.9, 50, seed=3), stop_tokens=[], logprobs=0)
    assert all(s.top == [] and s.logprob < 0 for o in drawn for s in o.logprobs)
    with pytest.raises(RocmlError, match="alternatives"):
        eng.generate(prompts, logprobs=33)
    with pytest.raises(RocmlError, match="alternatives"):
        eng.score(prompts, top=40)
