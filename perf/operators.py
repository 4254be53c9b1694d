"""Operators of verifying drafted tokens and of scoring, as cases that can be measured.

* ``attention``: softmax attention of a tree of drafted tokens over a paged cache.  A sequence brings its n nodes, whose keys and
  values already lie behind its context in its pages; a node sees the whole context (or a window of it) and, among the nodes, those
  that its row of bits names: its ancestors and itself.
* ``logprobs``: log probabilities of given tokens from rows of logits, with the rows' entropy and their most likely tokens.
* ``accept``: which nodes of every tree a sampler's tokens confirm, and the confirmed nodes' keys and values moved to the places
  behind the context where an ordinary step would have written them, in all layers.

``run`` computes them in their plain form unless ``own`` is set; then it calls the library.  Sizes are those of the catalog's
models (heads of 128, 8 key/value heads for 16 to 64 query heads, vocabularies of 151,936 and 32,768) and of the tests' small ones.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
PAGE = 64


def listed():
    return [
        # one user, a small model, a short draft over a short history: nothing but latency
        dict(name="tree 0.6b b1 n8", op="attention", dtype="bfloat16", nq=16, nkv=8, hd=128, seqs=1, few=8, many=8, short=701, long=701,
             window=0, keep=0, sink=False),
        # one user, a wide tree on the benchmark's model: as much arithmetic as bytes
        dict(name="tree 8b b1 n64", op="attention", dtype="bfloat16", nq=32, nkv=8, hd=128, seqs=1, few=64, many=64, short=4100, long=4100,
             window=0, keep=0, sink=False),
        # one user and a whole book
        dict(name="tree 8b b1 long", op="attention", dtype="bfloat16", nq=32, nkv=8, hd=128, seqs=1, few=16, many=16, short=100003, long=100003,
             window=0, keep=0, sink=False),
        # a busy server: trees and histories of all lengths side by side
        dict(name="tree 4b b32 ragged", op="attention", dtype="bfloat16", nq=32, nkv=8, hd=128, seqs=32, few=9, many=33, short=130, long=12100,
             window=0, keep=0, sink=False),
        # a window beside which the first positions stay visible, a sink in the denominator
        dict(name="tree window b8", op="attention", dtype="bfloat16", nq=32, nkv=8, hd=128, seqs=8, few=5, many=27, short=900, long=9000,
             window=4096, keep=4, sink=True),
        # the true 32-bit path
        dict(name="tree 32-bit b3", op="attention", dtype="float32", nq=16, nkv=8, hd=128, seqs=3, few=3, many=13, short=77, long=1337,
             window=0, keep=0, sink=False),
        # the one token that a user waits for, with the alternatives an interface shows
        dict(name="logprobs n1 top20", op="logprobs", dtype="float32", vocab=151936, rows=1, given=1, top=20, pad=0, masked=False),
        # a batch's step under a grammar that forbids most tokens
        dict(name="logprobs n64 masked", op="logprobs", dtype="float32", vocab=151936, rows=64, given=1, top=5, pad=0, masked=True),
        # a prompt scored token by token
        dict(name="logprobs n2047", op="logprobs", dtype="float32", vocab=151936, rows=2047, given=1, top=1, pad=0, masked=False),
        # candidate answers in half precision: rows that start off every boundary
        dict(name="logprobs bf16 odd", op="logprobs", dtype="bfloat16", vocab=32003, rows=333, given=4, top=8, pad=2, masked=False),
        # one user's draft, settled
        dict(name="accept 0.6b b1", op="accept", dtype="bfloat16", layers=28, nkv=8, hd=128, seqs=1, few=16, many=16, short=701, long=701, accepted=3),
        # a batch of large trees, settled
        dict(name="accept 4b b32", op="accept", dtype="bfloat16", layers=36, nkv=8, hd=128, seqs=32, few=20, many=64, short=100, long=1000, accepted=6),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attention", "attention", "attention", "logprobs", "logprobs", "accept"])
    if op == "attention":
        f32 = rng.random() < 0.2
        nkv = rng.choice([1, 2, 8]) if rng.random() < 0.3 else 8
        group = rng.choice([1, 2, 3, 4, 5, 8])
        hd = rng.choice([64, 128, 128, 128, 256])
        seqs, few = log_int(1, 4 if f32 else 40), log_int(1, 24)
        short = log_int(1, 2000 if f32 else 4000)
        case = dict(op=op, dtype="float32" if f32 else "bfloat16", nq=nkv * group, nkv=nkv, hd=hd, seqs=seqs, few=few,
                    many=few + rng.randrange(0, 41), short=short, long=short + log_int(1, 2000 if f32 else 110000), window=0, keep=0, sink=rng.random() < 0.25)
        if rng.random() < 0.25:
            case.update(window=log_int(64, 4096), keep=rng.choice([0, 4, 70]))
        # (never more than the largest listed case: the longest sequences give way)
        most = work(listed()[3])
        while work(case)["bytes"] > most["bytes"] / (4 if f32 else 1) or work(case)["flops"] > most["flops"] / (8 if f32 else 1) or \
                case["seqs"] * case["long"] * nkv * hd > 4e8:
            case["long"] = max(1, int(case["long"] * 0.7))
            case["short"] = min(case["short"], case["long"])
            case["seqs"] = max(1, int(case["seqs"] * 0.9))
        return case
    if op == "logprobs":
        half = rng.random() < 0.4
        vocab = rng.choice([151936, 32768, 50257, log_int(300, 160000)])
        return dict(op=op, dtype="bfloat16" if half else "float32", vocab=vocab, rows=log_int(1, 1000), given=rng.choice([1, 1, 2, 5]),
                    top=rng.choice([0, 1, 4, 20, 32]), pad=rng.choice([0, 0, 1, 64]), masked=rng.random() < 0.25)
    few, short = log_int(1, 40), log_int(1, 600)
    return dict(op=op, dtype=rng.choice(["bfloat16", "float32"]), layers=log_int(2, 36), nkv=rng.choice([1, 2, 8]), hd=rng.choice([16, 64, 128]),
                seqs=log_int(1, 24), few=few, many=few + rng.randrange(0, 25), short=short, long=short + log_int(1, 400), accepted=rng.randrange(0, 9))


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, in an order that mixes them."""
    v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]
    random.Random(n).shuffle(v)
    return v


def _sizes(case):
    """(nodes, context) of every sequence."""
    return _spread(case["few"], case["many"], case["seqs"]), _spread(case["short"], case["long"], case["seqs"])[::-1]


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    dtype = getattr(torch, case["dtype"])
    state = dict(case=case)

    def normal(shape, scale=1.0, dt=dtype):
        return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.bfloat16 if dt == torch.bfloat16 else torch.float32) * scale).to(dt)

    def ints(v):
        return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEVICE)

    if case["op"] == "logprobs":
        n, V = case["rows"], case["vocab"]
        # as a trained head leaves them: a broad bulk and a few tokens far above it, some of them nearly certain
        logits = normal((n, V + case["pad"]), 2.0)
        high = torch.randint(0, V, (n, 8), generator=g, device=DEVICE)
        logits.scatter_add_(1, high, (torch.rand((n, 8), generator=g, device=DEVICE) * 20).to(dtype))
        if case["masked"]:
            allowed = torch.rand((n, V + case["pad"]), generator=g, device=DEVICE) < 0.01
            allowed.scatter_(1, high, True)
            logits.masked_fill_(~allowed, -math.inf)
        ids = torch.randint(0, V, (n, case["given"]), generator=g, device=DEVICE)
        ids[:, 0] = torch.where(torch.rand(n, generator=g, device=DEVICE) < 0.7, high[:, 0], ids[:, 0])
        k = case["top"]
        state.update(logits=logits[:, :V], ids=ids.int(), logprobs=torch.empty((n, case["given"]), device=DEVICE), entropy=torch.empty(n, device=DEVICE),
                     top_logprobs=torch.empty((n, k), device=DEVICE), top_ids=torch.empty((n, k), dtype=torch.int32, device=DEVICE))
        return state

    def tree(rng, n, accepted):
        """Parents of n nodes (-1: the first) among which a chain of ``accepted`` nodes below the first is marked."""
        parents = [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)]
        chain = sorted(rng.sample(range(1, n), min(accepted, n - 1)))
        for above, node in zip([0] + chain, chain):
            parents[node] = above
        return parents, [0] + chain

    def bits(parents, words):
        """Rows of bits: a node's ancestors and itself."""
        rows = []
        for i, p in enumerate(parents):
            rows.append((1 << i) | (rows[p] if p >= 0 else 0))
        return np.frombuffer(b"".join(r.to_bytes(words * 4, "little") for r in rows), dtype=np.int32).reshape(len(parents), words)

    nodes, contexts = _sizes(case)
    B, words = case["seqs"], -(-max(nodes) // 32)
    pages = [-(-(c + n) // PAGE) for c, n in zip(contexts, nodes)]
    order = list(range(sum(pages) + 3))
    rng.shuffle(order)
    table = np.full((B + 2, max(pages) + 1), -1, dtype=np.int32)
    slots = rng.sample(range(B + 2), B)
    for slot, p in zip(slots, pages):
        table[slot, :p] = [order.pop() for _ in range(p)]
    trees = [tree(rng, n, case.get("accepted", n // 3)) for n in nodes]
    cu = np.concatenate([[0], np.cumsum(nodes)])
    state.update(table=ints(table), seq_slot=ints(slots), cu_q=ints(cu), kv_len=ints([c + n for c, n in zip(contexts, nodes)]),
                 visible=ints(np.concatenate([bits(p, words) for p, _ in trees])), max_nodes=max(nodes), max_len=max(c + n for c, n in zip(contexts, nodes)),
                 host=dict(nodes=nodes, contexts=contexts, slots=slots, table=table, trees=trees, cu=cu))
    n_pages, nkv, hd = sum(pages) + 3, case["nkv"], case["hd"]
    if case["op"] == "attention":
        depth = [bin(int.from_bytes(row.tobytes(), "little")).count("1") - 1 for row in np.concatenate([bits(p, words) for p, _ in trees])]
        state.update(positions=ints([contexts[b] + depth[t] for b in range(B) for t in range(cu[b], cu[b + 1])]),
                     q=normal((int(cu[-1]), case["nq"] * hd), 2.0), k=normal((n_pages, nkv, PAGE, hd)), v=normal((n_pages, nkv, PAGE, hd)),
                     out=torch.zeros((int(cu[-1]), case["nq"] * hd), dtype=dtype, device=DEVICE),
                     sink=normal((case["nq"],), 1.0, torch.float32) if case["sink"] else None)
        return state
    # the sampler confirms the marked chain, and below its last node draws a token that no child has
    tokens, sampled = [], []
    for parents, chain in trees:
        ids = [rng.randrange(151000) for _ in parents]
        draws = [rng.randrange(151000) for _ in parents]
        for above, node in zip(chain, chain[1:]):
            draws[above] = ids[node]
        draws[chain[-1]] = 151500
        tokens += ids
        sampled += draws
    state.update(parents=ints([p for parents, _ in trees for p in parents]), tokens=ints(tokens), sampled=ints(sampled),
                 k=normal((case["layers"], n_pages, nkv, PAGE, hd)), v=normal((case["layers"], n_pages, nkv, PAGE, hd)),
                 path=torch.empty((B, max(nodes)), dtype=torch.int32, device=DEVICE), counts=torch.empty(B, dtype=torch.int32, device=DEVICE),
                 next=torch.empty(B, dtype=torch.int32, device=DEVICE))
    state["host"].update(tokens=tokens, sampled=sampled)
    return state


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"attention": _attention, "logprobs": _logprobs, "accept": _accept}[case["op"]](state, case)


def _own(s, case):
    from rocml_b200 import kernels
    if case["op"] == "attention":
        kernels.attention_tree(s["q"], s["out"], s["k"], s["v"], s["table"], s["seq_slot"], s["cu_q"], s["kv_len"], s["visible"], case["seqs"],
                               s["max_nodes"], case["nq"], case["nkv"], case["hd"], case["hd"] ** -0.5, max_kv_len=s["max_len"],
                               positions=s["positions"], window=case["window"], keep=case["keep"], sink=s["sink"])
        return s["out"]
    if case["op"] == "logprobs":
        kernels.token_logprobs(s["logits"], s["ids"], s["logprobs"], s["entropy"], s["top_logprobs"], s["top_ids"])
        return s["logprobs"], s["entropy"], s["top_logprobs"], s["top_ids"]
    kernels.tree_accept(s["tokens"], s["parents"], s["visible"], s["sampled"], s["cu_q"], case["seqs"], s["path"], s["counts"], s["next"],
                        seq_slot=s["seq_slot"], kv_len=s["kv_len"], block_table=s["table"], k=s["k"], v=s["v"])
    return s["path"], s["counts"], s["next"], s["k"], s["v"]


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _rows(s):
    """Sequence and place within its tree of every node."""
    cu = s["cu_q"].long()
    t = torch.arange(s["visible"].shape[0], device=DEVICE)
    seq = torch.bucketize(t, cu[1:], right=True)
    return seq, t - cu[seq]


def _unpacked(visible):
    return ((visible.unsqueeze(-1) >> torch.arange(32, device=DEVICE, dtype=torch.int32)) & 1).bool().flatten(1)


def _attention(s, case):
    B, N, nq, nkv, hd = case["seqs"], s["max_nodes"], case["nq"], case["nkv"], case["hd"]
    seq, node = _rows(s)
    ctx = (s["kv_len"] - (s["cu_q"][1:] - s["cu_q"][:-1])).long()
    L = -(-s["max_len"] // PAGE) * PAGE
    pages = s["table"][s["seq_slot"].long(), :L // PAGE].long().clamp_min(0)
    k, v = (x[pages].float().permute(0, 2, 1, 3, 4).reshape(B, nkv, L, hd) for x in (s["k"], s["v"]))
    q = torch.zeros((B, N, nq, hd), device=DEVICE)
    q[seq, node] = s["q"].float().view(-1, nq, hd)
    place = torch.arange(L, device=DEVICE)
    v = v * (place < s["kv_len"].long().unsqueeze(1)).view(B, 1, L, 1)
    # which places a node sees: the context (its window and the first ones kept), and behind it the nodes its bits name
    sees = torch.zeros((B, N, L), dtype=torch.bool, device=DEVICE)
    context = place < ctx[seq].unsqueeze(1)
    if case["window"]:
        context &= (place > s["positions"].unsqueeze(1) - case["window"]) | (place < case["keep"])
    bits = _unpacked(s["visible"])
    at = (place - ctx[seq].unsqueeze(1))
    sees[seq, node] = context | ((at >= 0) & (at < bits.shape[1]) & bits.gather(1, at.clamp(0, bits.shape[1] - 1)))
    q = q.permute(0, 2, 1, 3).reshape(B, nkv, nq // nkv * N, hd)
    scores = (q @ k.transpose(2, 3)).view(B, nkv, nq // nkv, N, L) * hd ** -0.5
    scores = scores.masked_fill(~sees.view(B, 1, 1, N, L), -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"].view(1, nkv, nq // nkv, 1, 1) - top)
    o = (e / total.clamp_min(1e-30)).view(B, nkv, nq // nkv * N, L) @ v
    return o.view(B, nq, N, hd).transpose(1, 2)[seq, node].reshape(-1, nq * hd).to(s["q"].dtype)


def _logprobs(s, case):
    x, V = s["logits"].float(), case["vocab"]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    below = torch.where(e > 0, (x - top) * e, 0.0)
    entropy = log_total[:, 0] - below.sum(1) / total[:, 0]
    given = x.gather(1, s["ids"].long()) - top - log_total
    # largest first, equal ones by their place: whole numbers that order like (value, -place)
    raw = (x + 0.0).view(torch.int32).long()
    order = torch.where(raw < 0, raw ^ 0x7FFFFFFF, raw) * 2 ** 32 + (V - 1 - torch.arange(V, device=DEVICE))
    best = V - 1 - (torch.topk(order, case["top"], dim=1).values & 0xFFFFFFFF)
    return given, entropy, x.gather(1, best) - top - log_total, best.int()


def _accept(s, case):
    B, N = case["seqs"], s["max_nodes"]
    seq, node = _rows(s)
    parents, T = s["parents"].long(), s["parents"].numel()
    above = s["cu_q"].long()[seq] + parents.clamp_min(0)
    like = (parents >= 0) & (s["tokens"] == s["sampled"][above])
    # of several children with the drawn token the first one counts
    flat = torch.arange(T, device=DEVICE)
    first = torch.full((T,), T, device=DEVICE).scatter_reduce(0, torch.where(like, above, flat), torch.where(like, flat, T), "amin")
    like = torch.where(parents >= 0, like & (first[above] == flat), node == 0)
    bits = _unpacked(s["visible"])
    table = torch.zeros((B, bits.shape[1]), dtype=torch.bool, device=DEVICE)
    table[seq, node] = like
    kept = (table[seq] | ~bits).all(1)
    depth = bits.sum(1) - 1
    counts = torch.zeros(B, dtype=torch.int32, device=DEVICE).index_add_(0, seq, kept.int())
    path = torch.full((B, N), -1, dtype=torch.int32, device=DEVICE)
    path[seq[kept], depth[kept]] = node[kept].int()
    last = path.gather(1, counts.long().unsqueeze(1) - 1)[:, 0]
    nxt = s["sampled"][s["cu_q"][:-1].long() + last]
    # every confirmed node's keys and values to the place that its depth gives it
    slot = s["seq_slot"].long()[seq[kept]]
    ctx = (s["kv_len"] - (s["cu_q"][1:] - s["cu_q"][:-1])).long()[seq[kept]]
    src, dst = ctx + node[kept], ctx + depth[kept]
    sp, dp = s["table"][slot, src // PAGE].long(), s["table"][slot, dst // PAGE].long()
    k, v = s["k"], s["v"]
    k[:, dp, :, dst % PAGE] = k[:, sp, :, src % PAGE]
    v[:, dp, :, dst % PAGE] = v[:, sp, :, src % PAGE]
    return path, counts, nxt, k, v


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "logprobs":
        n, V = case["rows"], case["vocab"]
        return {"bytes": n * V * size + n * (8 * case["given"] + 4 + 8 * case["top"]), "flops": 5 * n * V}
    nodes, contexts = _sizes(case)
    if case["op"] == "attention":
        nq, nkv, hd, w = case["nq"], case["nkv"], case["hd"], case["window"]
        read = [(min(c, w + case["keep"]) if w else c) for c in contexts]
        nbytes = sum(r + n for r, n in zip(read, nodes)) * 2 * nkv * hd * size + sum(nodes) * (2 * nq * hd * size + 4 * -(-max(nodes) // 32))
        return {"bytes": nbytes, "flops": 4 * nq * hd * sum(n * (r + 1) for r, n in zip(read, nodes))}
    moved = sum(min(case["accepted"], n - 1) for n in nodes)
    return {"bytes": moved * case["layers"] * case["nkv"] * case["hd"] * size * 4 + 20 * sum(nodes), "flops": sum(nodes)}


# ---- the same by the definitions, in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        given, entropy, alternatives, best = [], [], [], []
        for x, ids in zip(s["logits"].split(64), s["ids"].split(64)):
            x = x.double()
            logp = x - torch.logsumexp(x, 1, keepdim=True)
            given.append(logp.gather(1, ids.long()))
            entropy.append(-(logp.exp() * logp.clamp_min(-1e300)).sum(1))
            value, place = torch.sort(logp, dim=1, descending=True, stable=True)
            alternatives.append(value[:, :case["top"]])
            best.append(place[:, :case["top"]].int())
        return tuple(torch.cat(v) for v in (given, entropy, alternatives, best))
    h = s["host"]
    if case["op"] == "attention":
        out = torch.zeros((s["q"].shape[0], case["nq"], case["hd"]), dtype=torch.float64, device=DEVICE)
        group = case["nq"] // case["nkv"]
        for b, (n, c, slot, (parents, _)) in enumerate(zip(h["nodes"], h["contexts"], h["slots"], h["trees"])):
            pages = torch.tensor(h["table"][slot, :-(-(c + n) // PAGE)], device=DEVICE).long()
            hidden = np.ones((n, c + n), dtype=bool)
            for i in range(n):
                up, depth = i, 0
                while up >= 0:
                    hidden[i, c + up] = False
                    up, depth = parents[up], depth + 1
                first = max(0, c + depth - 1 - case["window"] + 1) if case["window"] else 0
                hidden[i, min(first, c):c] = False
                hidden[i, :min(c, case["keep"])] &= not case["window"]
            hidden = torch.tensor(hidden, device=DEVICE)
            for head in range(case["nq"]):
                k, v = (x[pages, head // group].reshape(-1, case["hd"])[:c + n].double() for x in (s["k"], s["v"]))
                scores = s["q"][h["cu"][b]:h["cu"][b + 1], head * case["hd"]:(head + 1) * case["hd"]].double() @ k.t() / math.sqrt(case["hd"])
                scores = scores.masked_fill(hidden, -math.inf)
                bottom = torch.logsumexp(scores, 1)
                if s["sink"] is not None:
                    bottom = torch.logaddexp(bottom, s["sink"][head].double())
                out[h["cu"][b]:h["cu"][b + 1], head] = torch.exp(scores - bottom.unsqueeze(1)) @ v
        return out.reshape(-1, case["nq"] * case["hd"])
    paths, counts, nxt = torch.full((case["seqs"], s["max_nodes"]), -1, dtype=torch.int32), [], []
    k, v = s["k"].clone(), s["v"].clone()
    for b, (c, slot, (parents, _)) in enumerate(zip(h["contexts"], h["slots"], h["trees"])):
        first, here, count = int(h["cu"][b]), 0, 0
        while here is not None:
            paths[b, count] = here
            (p, i), (sp, si) = divmod(c + count, PAGE), divmod(c + here, PAGE)
            p, sp = int(h["table"][slot, p]), int(h["table"][slot, sp])
            k[:, p, :, i], v[:, p, :, i] = s["k"][:, sp, :, si], s["v"][:, sp, :, si]
            count, drawn = count + 1, h["sampled"][first + here]
            here = next((j for j, up in enumerate(parents) if up == here and h["tokens"][first + j] == drawn), None)
        counts.append(count)
        nxt.append(drawn)
    return paths, torch.tensor(counts, dtype=torch.int32), torch.tensor(nxt, dtype=torch.int32), k.double(), v.double()
