"""Attention over trees of drafted tokens, and settling such trees, against plain 64-bit forms."""
import math
import random

import pytest
import torch

import plain_tree
from plain_tree import Trees, as_words

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# sequences as (context, nodes): none, one and many keys; nodes that end a page, begin one, span two to four
SIZES = {
    "one": [(0, 1)],
    "few": [(5, 3), (0, 9), (64, 1), (63, 1), (63, 2), (128, 64)],
    "ragged": [(700, 33), (1, 1), (190, 70), (0, 130), (64, 5)],
    "long": [(2100, 17), (3, 40)],
}


def bound(want, mass, dtype, tc):
    """Weights, sums and results are 32-bit: their error is within 2e-5 of sum(weight |value|) (scores up to about 30 in base e with an error of
    2^-24 of themselves, sums of up to 2,100 terms).  A bfloat16 result is rounded once more (half a step, 2^-8 of itself at most);
    the tensor-core kernel also rounds every weight to bfloat16 (2^-8 of it at most, numerator and not denominator)."""
    b = 2e-5 * mass + 1e-7
    if dtype == torch.bfloat16:
        b = b + 2 ** -8 * want.abs()
        if tc:
            b = b + 2 ** -8 * mass
    return b


def call(t, window=0, keep=0, sink=None, softcap=0.0, scale=None, max_len=True, out=None, **ints):
    from rocml_b200 import kernels
    d = dict(t.ints(DEV), **ints)
    q = t.q.to(DEV)
    out = torch.full_like(q, 7.0) if out is None else out
    n = max([1] + [n for _, n in t.sizes])
    kernels.attention_tree(q, out, t.k[0].to(DEV), t.v[0].to(DEV), d["block_table"], d["seq_slot"], d["cu_q"], d["kv_len"], d["visible"],
                           len(t.sizes), n, t.nq, t.nkv, t.hd, t.hd ** -0.5 if scale is None else scale,
                           max_kv_len=max(c + n for c, n in t.sizes) if max_len else None,
                           positions=t.positions.to(DEV), window=window, keep=keep, sink=sink, softcap=softcap)
    kernels.check_status(DEV)
    return out


def check(t, dtype, out, **options):
    want, mass = plain_tree.attention(t, t.hd ** -0.5, **options)
    err = (out.double().cpu() - want).abs()
    over = (err - bound(want, mass, dtype, t.hd in (64, 128, 256))).max().item()
    assert over <= 0, (over, err.max().item())


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 64), (8, 2, 128), (3, 3, 128), (6, 2, 256), (5, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_tree(sizes, nq, nkv, hd, dtype):
    t = Trees(len(sizes) + nq, SIZES[sizes], nq, nkv, hd, dtype)
    check(t, dtype, call(t))


@pytest.mark.parametrize("hd", [1, 16, 30, 48, 80, 192, 320, 512])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_tree_other_head_sizes(hd, dtype):
    t = Trees(hd, [(70, 9), (0, 3)], 4, 2, hd, dtype)
    check(t, dtype, call(t))


@pytest.mark.parametrize("window,keep", [(1, 0), (5, 0), (64, 3), (100, 70), (3000, 4)])
@pytest.mark.parametrize("dtype,hd", [(torch.float32, 48), (torch.bfloat16, 128), (torch.bfloat16, 64)])
def test_attention_tree_windows(window, keep, dtype, hd):
    t = Trees(window, [(700, 33), (3, 5), (128, 20), (2050, 12)], 4, 2, hd, dtype)
    check(t, dtype, call(t, window=window, keep=keep), window=window, keep=keep)


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 128)])
def test_attention_tree_sinks_and_soft_cap(dtype, hd):
    t = Trees(5, [(300, 20), (0, 2), (1500, 7)], 4, 2, hd, dtype)
    sinks = torch.tensor([1.0, -3.0, 8.0, -math.inf])
    check(t, dtype, call(t, sink=sinks.to(DEV)), sinks=sinks)
    check(t, dtype, call(t, sink=2.5), sinks=torch.full((4,), 2.5))
    check(t, dtype, call(t, softcap=15.0), softcap=15.0)
    check(t, dtype, call(t, softcap=15.0, sink=sinks.to(DEV), window=200, keep=5), softcap=15.0, sinks=sinks, window=200, keep=5)


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 32), (torch.bfloat16, 128)])
def test_attention_tree_rows_that_see_nothing_and_any_bits(dtype, hd):
    """Bits of any pattern; an empty row without a context is zero; bits beyond the tree mean nothing."""
    t = Trees(3, [(0, 6), (40, 6), (0, 90)], 4, 2, hd, dtype)
    rng = random.Random(4)
    rows = [rng.getrandbits(96) for _ in range(t.cu[-1])]
    rows[0] = rows[7] = rows[20] = 0
    rows[1] = 1 << 80                                   # (a node that its tree of six does not have)
    t.visible = as_words(rows, 3)
    out = call(t)
    assert (out[0] == 0).all() and (out[1] == 0).all() and (out[20] == 0).all()
    check_rows = Trees.__new__(Trees)
    check_rows.__dict__.update(t.__dict__)
    cut = [r & ((1 << n) - 1) for r, n in zip(rows, [6] * 12 + [90] * 90)]
    check_rows.visible = as_words(cut, 3)
    check(check_rows, dtype, out)


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 256)])
def test_attention_tree_hidden_places_may_hold_anything(dtype, hd):
    """NaN and infinities in places that a row does not see (behind the sequence's end, below its window, siblings) do not reach it."""
    t = Trees(6, [(130, 10), (400, 30)], 4, 2, hd, dtype)
    want = call(t, window=100, keep=3)
    for b, (c, n) in enumerate(t.sizes):
        for p in list(range(c + n, -(-(c + n) // 64) * 64)) + list(range(3, c - 100)):
            page, at = t.place(b, p)
            t.k[0, page, :, at] = float("nan") if p % 2 else float("inf")
            t.v[0, page, :, at] = float("inf") if p % 3 else float("nan")
    assert torch.equal(call(t, window=100, keep=3), want)
    # a node's own value is not finite: the rows that see it show it, the others do not
    c, n = t.sizes[1]
    page, at = t.place(1, c + 3)
    t.v[0, page, :, at, 5] = float("inf")
    out = call(t, window=100, keep=3)
    sees = torch.tensor([plain_tree.bit(t.visible, r, 3) for r in range(t.cu[1], t.cu[2])], dtype=torch.bool)
    assert sees.any() and not sees.all()
    assert not torch.isfinite(out[t.cu[1]:][sees][:, 5]).any()
    assert torch.equal(out[:t.cu[1]], want[:t.cu[1]]) and torch.equal(out[t.cu[1]:][~sees], want[t.cu[1]:][~sees])


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 128)])
def test_attention_tree_leaves_other_rows_alone(dtype, hd):
    """Padding sequences (slot -1, no rows), sequences that say less than their tree or more than their row of the table, rows behind the
    last sequence: nothing is written there, and the others are right.  (Not the same bits: where a sequence's keys are cut among blocks depends on
    the other sequences, and the order of 32-bit sums on that.)"""
    t = Trees(8, [(100, 4), (50, 6), (30, 3), (20, 2)], 4, 2, hd, dtype)
    want, mass = plain_tree.attention(t, hd ** -0.5)
    right = lambda out, n: ((out[:n].double().cpu() - want[:n]).abs() <= bound(want, mass, dtype, hd in (64, 128, 256))[:n]).all()
    slots, lens = list(t.slots), [c + n for c, n in t.sizes]
    slots[1] = -1
    lens[2] = 2
    lens[3] = 64 * t.table.shape[1] + 1
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    out = call(t, seq_slot=i32(slots), kv_len=i32(lens))
    assert right(out, 4) and (out[4:] == 7.0).all()
    out = call(t, cu_q=i32([0, 4, 10, 10, 10]))          # the last two bring nothing
    assert right(out, 10) and (out[10:] == 7.0).all()


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 48), (torch.bfloat16, 128), (torch.bfloat16, 64)])
def test_attention_tree_strided_rows(dtype, hd):
    """q and out as columns of wider rows; rows off every alignment take the plain kernel."""
    from rocml_b200 import kernels
    t = Trees(9, [(333, 21), (12, 5)], 4, 2, hd, dtype)
    want = call(t)
    d = t.ints(DEV)
    for left, right in ((8, 16), (3, 2)):
        T, W = t.q.shape
        q = torch.full((T, left + W + right), float("nan"), dtype=dtype, device=DEV)
        out = torch.full_like(q, 7.0)
        q[:, left:left + W] = t.q.to(DEV)
        kernels.attention_tree(q[:, left:left + W], out[:, left:left + W], t.k[0].to(DEV), t.v[0].to(DEV), d["block_table"], d["seq_slot"],
                               d["cu_q"], d["kv_len"], d["visible"], 2, 21, 4, 2, hd, hd ** -0.5, max_kv_len=354)
        kernels.check_status(DEV)
        check(t, dtype, out[:, left:left + W])
        if left == 8:
            assert torch.equal(out[:, left:left + W], want)
        assert (out[:, :left] == 7).all() and (out[:, left + W:] == 7).all()


def test_attention_tree_many_sequences_and_many_tiles():
    """More sequences than a warp counts at once, more tiles than blocks run at once."""
    t = Trees(10, [(i % 7 * 13, 1 + i % 4) for i in range(150)], 2, 1, 64, torch.bfloat16)
    check(t, torch.bfloat16, call(t))
    t = Trees(11, [(200, 256), (10, 250)], 40, 4, 64, torch.bfloat16)
    check(t, torch.bfloat16, call(t))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_tree_in_a_graph_and_on_another_stream(dtype):
    """The same bits eagerly, captured and replayed on new contents, and beside itself on two streams; twice the same."""
    from rocml_b200 import kernels
    t, u = (Trees(s, [(900, 20), (77, 9)], 8, 2, 128, dtype) for s in (12, 13))
    want_t, want_u = call(t), call(u)
    assert torch.equal(call(t), want_t)
    d = t.ints(DEV)
    q, k, v, out = t.q.to(DEV), t.k[0].to(DEV), t.v[0].to(DEV), torch.zeros_like(want_t)
    args = lambda q, k, v, out, d: kernels.attention_tree(q, out, k, v, d["block_table"], d["seq_slot"], d["cu_q"], d["kv_len"], d["visible"], 2, 20,
                                                          8, 2, 128, 128 ** -0.5, max_kv_len=920)
    args(q, k, v, out, d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        args(q, k, v, out, d)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want_t)
    for a, b in ((q, u.q), (k, u.k[0]), (v, u.v[0])):
        a.copy_(b)
    for name, x in u.ints(DEV).items():
        d[name].copy_(x)
    graph.replay()
    assert torch.equal(out, want_u)
    e, outs = [t.ints(DEV), u.ints(DEV)], [torch.zeros_like(out) for _ in range(2)]
    tensors = [[x.to(DEV) for x in (s.q, s.k[0], s.v[0])] for s in (t, u)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, x, o, ints in zip(streams, tensors, outs, e):
            with torch.cuda.stream(s):
                args(*x, o, ints)
    torch.cuda.synchronize()
    kernels.check_status(DEV)
    assert torch.equal(outs[0], want_t) and torch.equal(outs[1], want_u)


def test_attention_tree_behind_32_bit_offsets():
    """A cache of 2^33 bytes whose last pages hold the sequence."""
    from rocml_b200 import kernels
    t = Trees(14, [(100, 8)], 4, 2, 128, torch.bfloat16)
    want = call(t)
    pages = 2 ** 33 // (2 * 64 * 128 * 2) + 4
    k, v = (torch.empty((pages, 2, 64, 128), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    d = t.ints(DEV)
    moved = torch.where(t.table >= 0, pages - 1 - t.table, t.table)
    for p in set(int(x) for x in t.table.reshape(-1) if x >= 0):
        k[pages - 1 - p], v[pages - 1 - p] = t.k[0, p].to(DEV), t.v[0, p].to(DEV)
    out = torch.zeros_like(want)
    kernels.attention_tree(t.q.to(DEV), out, k, v, moved.to(DEV), d["seq_slot"], d["cu_q"], d["kv_len"], d["visible"], 1, 8, 4, 2, 128, 128 ** -0.5,
                           max_kv_len=108)
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_attention_tree_gives_the_same_bits_every_time(dtype, hd):
    """Ragged batches whose blocks take pieces of several sequences, two hundred times over under full load of the memory."""
    g = torch.Generator(DEV).manual_seed(1)
    contexts, nodes = [4 + 277 * i for i in range(19)], [2 + i * 7 % 13 for i in range(19)]
    from rocml_b200 import kernels
    pages = [-(-(c + n) // 64) for c, n in zip(contexts, nodes)]
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(2)).tolist()
    table = torch.full((19, max(pages)), -1, dtype=torch.int32)
    for b, p in enumerate(pages):
        table[b, :p] = torch.tensor([order.pop() for _ in range(p)])
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    rng = random.Random(3)
    visible = torch.cat([plain_tree.bits_of(plain_tree.random_parents(rng, n), 1) for n in nodes]).to(DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    k, v = (torch.randn((sum(pages), 8, 64, hd), generator=g, device=DEV).to(dtype) for _ in range(2))
    q = (torch.randn((cu[-1], 40 * hd), generator=g, device=DEV) * 2).to(dtype)
    out, first = torch.zeros_like(q), None
    args = (table.to(DEV), i32(list(range(19))), i32(cu), i32([c + n for c, n in zip(contexts, nodes)]), visible)
    for _ in range(200):
        out.zero_()
        kernels.attention_tree(q, out, k, v, *args, 19, max(nodes), 40, 8, hd, hd ** -0.5, max_kv_len=5200)
        first = out.clone() if first is None else first
        assert torch.equal(out, first)
    kernels.check_status(DEV)


# ---- settling a tree ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,hd,layers,nkv", [(torch.bfloat16, 128, 3, 2), (torch.float32, 48, 2, 1), (torch.bfloat16, 30, 1, 3), (torch.float32, 3, 2, 2)])
@pytest.mark.parametrize("sizes", ["one", "few", "ragged"])
def test_tree_accept(dtype, hd, layers, nkv, sizes):
    from rocml_b200 import kernels
    t = Trees(21, SIZES[sizes], nkv, nkv, hd, dtype, layers=layers)
    rng = random.Random(5)
    B, most = len(t.sizes), max(n for _, n in t.sizes)
    tokens = [[rng.randrange(2) for _ in p] for p in t.parents]          # (equal children are common)
    sampled = [[rng.randrange(2) for _ in p] for p in t.parents]
    k, v = t.k.clone(), t.v.clone()
    paths, counts, nxt = torch.full((B, most + 2), -1, dtype=torch.int32), [], []
    for b, (c, n) in enumerate(t.sizes):
        path, drawn = plain_tree.accept(t.parents[b], tokens[b], sampled[b])
        paths[b, :len(path)] = torch.tensor(path)
        counts.append(len(path))
        nxt.append(drawn)
        for d, node in enumerate(path):
            (p, i), (sp, si) = t.place(b, c + d), t.place(b, c + node)
            k[:, p, :, i], v[:, p, :, i] = t.k[:, sp, :, si], t.v[:, sp, :, si]
    assert sizes == "one" or any(x > 1 for x in counts)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    d = t.ints(DEV)
    got_k, got_v = t.k.to(DEV), t.v.to(DEV)
    path, count, drawn = torch.full((B, most + 2), 9, dtype=torch.int32, device=DEV), i32([9] * B), i32([9] * B)
    flat = lambda x: i32([y for s in x for y in s])
    kernels.tree_accept(flat(tokens), flat(t.parents), d["visible"], flat(sampled), d["cu_q"], B, path, count, drawn, seq_slot=d["seq_slot"],
                        kv_len=d["kv_len"], block_table=d["block_table"], k=got_k, v=got_v)
    assert torch.equal(path.cpu(), paths) and count.tolist() == counts and drawn.tolist() == nxt
    assert torch.equal(got_k.cpu(), k) and torch.equal(got_v.cpu(), v)
    # without a cache the same path; a sequence of a slot below 0 stays as it is
    path2, count2 = torch.full_like(path, 9), i32([9] * B)
    slots = d["seq_slot"].clone()
    slots[0] = -1
    kernels.tree_accept(flat(tokens), flat(t.parents), d["visible"], flat(sampled), d["cu_q"], B, path2, count2, drawn, seq_slot=slots)
    assert (path2[0] == 9).all() and count2[0] == 9 and torch.equal(path2[1:], path[1:]) and torch.equal(count2[1:], count[1:])


def test_tree_accept_a_whole_chain_of_256():
    from rocml_b200 import kernels
    t = Trees(22, [(1000, 256)], 1, 1, 16, torch.bfloat16)
    parents = list(range(-1, 255))
    t.visible = plain_tree.bits_of(parents, 8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    d = t.ints(DEV)
    k, v = t.k.to(DEV), t.v.to(DEV)
    path, count, drawn = torch.zeros((1, 256), dtype=torch.int32, device=DEV), i32([0]), i32([0])
    kernels.tree_accept(i32(list(range(256))), i32(parents), d["visible"], i32(list(range(1, 257))), d["cu_q"], 1, path, count, drawn,
                        seq_slot=d["seq_slot"], kv_len=d["kv_len"], block_table=d["block_table"], k=k, v=v)
    assert path[0].tolist() == list(range(256)) and count.item() == 256 and drawn.item() == 256
    assert torch.equal(k.cpu(), t.k) and torch.equal(v.cpu(), t.v)


@pytest.mark.parametrize("blocks", [0, 2, 5, 7, 16])
@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 64), (8, 2, 128), (6, 2, 256), (16, 1, 64)])
@pytest.mark.parametrize("sizes", list(SIZES))
def test_attention_tree_blocks_of_a_cluster(blocks, nq, nkv, hd, sizes, monkeypatch):
    """However many blocks share a sequence's pages, and joining by either way."""
    from rocml_b200 import kernels
    monkeypatch.setattr(kernels, "tree_cluster", lambda *a: blocks)
    kernels._tree_plan.cache_clear()
    try:
        t = Trees(blocks + nq, SIZES[sizes], nq, nkv, hd, torch.bfloat16)
        check(t, torch.bfloat16, call(t))
        sinks = torch.linspace(-3.0, 2.0, nq)
        options = dict(window=150, keep=20, softcap=8.0)
        first = call(t, sink=sinks.to(DEV), **options)
        check(t, torch.bfloat16, first, sinks=sinks, **options)
        assert all(torch.equal(first, call(t, sink=sinks.to(DEV), **options)) for _ in range(20))
    finally:
        kernels._tree_plan.cache_clear()
