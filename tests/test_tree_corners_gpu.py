"""Trees of drafted tokens and scoring at the edges of what a call allows: keys that are not finite, positions past the sequence's last place,
sequences without nodes, rows without enough finite logits."""
import math

import pytest
import torch

import plain_tree
from plain_tree import Trees
from test_tree_gpu import DEV, bound, call, check

pytestmark = pytest.mark.gpu


@pytest.fixture
def cluster_of(monkeypatch):
    """Sets how many blocks share a sequence's pages in the tensor-core kernel (0: equal shares and a second kernel; None: by the rule)."""
    from rocml_b200 import kernels

    def choose(blocks):
        if blocks is not None:
            monkeypatch.setattr(kernels, "tree_cluster", lambda *a: blocks)
        kernels._tree_plan.cache_clear()
    yield choose
    kernels._tree_plan.cache_clear()


@pytest.mark.parametrize("dtype,nq,nkv,hd,blocks", [(torch.bfloat16, q, n, h, b) for q, n, h in ((8, 2, 128), (16, 1, 64), (6, 2, 256)) for b in (0, 2, 7, 16)]
                         + [(torch.float32, 4, 2, 64, None), (torch.bfloat16, 4, 2, 48, None)])
def test_keys_that_are_not_finite_reach_the_rows_that_see_them(dtype, nq, nkv, hd, blocks, cluster_of):
    """Pages of nothing but NaN keys, whichever block they fall to: NaN in the rows that see them, the same bits in the others."""
    cluster_of(blocks)
    t = Trees(41 + hd, [(700, 33), (640, 128), (190, 9)], nq, nkv, hd, dtype)
    want = call(t)
    assert torch.isfinite(want).all()
    kept = t.k.clone()
    for places in ([192], range(0, 384, 64)):          # inside the first sequence's context, one page and half of them: all its rows
        for p in places:
            t.k[0, t.place(0, p)[0]] = math.nan
        out = call(t)
        assert torch.isnan(out[:t.cu[1]]).all() and torch.equal(out[t.cu[1]:], want[t.cu[1]:])
        t.k = kept.clone()
    t.k[0, t.place(1, 704)[0]] = math.nan              # the second sequence's nodes 64 to 127: themselves
    out = call(t)
    hit = slice(t.cu[1] + 64, t.cu[2])
    assert torch.isnan(out[hit]).all()
    assert torch.equal(out[:hit.start], want[:hit.start]) and torch.equal(out[hit.stop:], want[hit.stop:])


@pytest.mark.parametrize("window,keep", [(1, 0), (64, 3), (100, 70), (300, 0)])
@pytest.mark.parametrize("dtype,hd", [(torch.float32, 48), (torch.bfloat16, 128), (torch.bfloat16, 64)])
def test_positions_past_the_sequences_last_place(window, keep, dtype, hd):
    """A window goes by a node's position, wherever that is: none of the context may be left of it."""
    t = Trees(window + hd, [(700, 33), (3, 5), (128, 20), (2050, 12)], 4, 2, hd, dtype)
    t.positions = t.positions + torch.arange(t.cu[-1], dtype=torch.int32) * 37 % 250
    check(t, dtype, call(t, window=window, keep=keep), window=window, keep=keep)


def test_a_sequence_without_nodes_has_nothing_confirmed():
    from rocml_b200 import kernels
    t = Trees(5, [(30, 3), (64, 1), (10, 4)], 1, 1, 16, torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    d = t.ints(DEV)
    cu, lens = i32([0, 3, 3, 7]), i32([33, 64, 14])
    visible = torch.cat([plain_tree.bits_of(p, 1) for p in ([-1, 0, 1], [-1, 0, 0, 1])]).to(DEV)
    k, v = t.k.to(DEV), t.v.to(DEV)
    path, counts, drawn = torch.full((3, 5), 9, dtype=torch.int32, device=DEV), i32([9] * 3), i32([9] * 3)
    kernels.tree_accept(i32([4, 5, 6, 4, 8, 5, 7]), i32([-1, 0, 1, -1, 0, 0, 1]), visible, i32([5, 6, 1, 5, 3, 2, 0]), cu, 3, path, counts, drawn,
                        seq_slot=d["seq_slot"], kv_len=lens, block_table=d["block_table"], k=k, v=v)
    assert path.tolist() == [[0, 1, 2, -1, -1], [-1] * 5, [0, 2, -1, -1, -1]] and counts.tolist() == [3, 0, 2] and drawn.tolist() == [1, -1, 2]


@pytest.mark.parametrize("V,top", [(1, 1), (3, 3), (3000, 5), (40000, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alternatives_of_a_row_that_holds_nan_are_nan(V, top, dtype):
    """However few of its logits are numbers."""
    from rocml_b200 import kernels
    x = torch.full((4, V), math.nan, dtype=dtype)
    x[1, :V // 2] = 1.0
    x[2, 1:] = torch.randn(V - 1, generator=torch.Generator().manual_seed(V)).to(dtype)
    x[3] = -math.inf
    values, ids = torch.full((4, top), 9.0, device=DEV), torch.full((4, top), 9, dtype=torch.int32, device=DEV)
    kernels.token_logprobs(x.to(DEV), None, None, None, values, ids)
    assert torch.isnan(values[:3]).all() and torch.isneginf(values[3]).all()
    assert (ids[0] == -1).all() and ids[3].tolist() == list(range(top)) and ((ids >= -1) & (ids < V)).all()


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_a_call_without_a_single_node(dtype, hd):
    from rocml_b200 import kernels
    t = Trees(6, [(70, 2), (5, 3)], 4, 2, hd, dtype)
    d = t.ints(DEV)
    q, out = torch.zeros((0, 4 * hd), dtype=dtype, device=DEV), torch.full((5, 4 * hd), 7.0, dtype=dtype, device=DEV)
    kernels.attention_tree(q, out, t.k[0].to(DEV), t.v[0].to(DEV), d["block_table"], d["seq_slot"], torch.zeros_like(d["cu_q"]), d["kv_len"],
                           d["visible"][:0], 2, 1, 4, 2, hd, 0.1)
    kernels.check_status(DEV)
    assert (out == 7).all()


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 48), (torch.bfloat16, 128)])
def test_as_many_kept_places_as_an_integer_holds(dtype, hd):
    """More than the context has: the whole of it is kept, as without a window."""
    t = Trees(7, [(700, 33), (3, 5), (128, 20)], 4, 2, hd, dtype)
    for keep in (2 ** 31 - 1, 2 ** 31 - 64, 2 ** 20):
        check(t, dtype, call(t, window=5, keep=keep), window=5, keep=keep)
    check(t, dtype, call(t, window=2 ** 31 - 1, keep=2 ** 31 - 1))


@pytest.mark.parametrize("sizes", [[(70, 9), (0, 3)], [(1500, 17), (64, 40)]])
@pytest.mark.parametrize("dtype,nq,hd", [(torch.float32, 16, 32), (torch.bfloat16, 9, 64), (torch.bfloat16, 32, 128), (torch.bfloat16, 17, 256), (torch.bfloat16, 20, 512)])
def test_keys_and_values_in_one_tensor(sizes, dtype, nq, hd):
    """A latent that serves as both, read by many heads: attention over it, and the confirmed path's rows moved once."""
    from rocml_b200 import kernels
    t = Trees(nq, sizes, nq, 1, hd, dtype, layers=2)
    t.v = t.k
    d = t.ints(DEV)
    both = t.k.to(DEV)
    q = t.q.to(DEV)
    out = torch.full_like(q, 7.0)
    kernels.attention_tree(q, out, both[0], both[0], d["block_table"], d["seq_slot"], d["cu_q"], d["kv_len"], d["visible"], 2, max(n for _, n in sizes), nq, 1,
                           hd, hd ** -0.5, max_kv_len=max(c + n for c, n in sizes), positions=t.positions.to(DEV), window=200)
    kernels.check_status(DEV)
    check(t, dtype, out, window=200)
    tokens = [list(range(n)) for _, n in sizes]
    sampled = [[max([j for j, up in enumerate(p) if up == i], default=0) for i in range(len(p))] for p in t.parents]       # (the last child)
    want, i32 = t.k.clone(), lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    moved = 0
    for b, (c, n) in enumerate(sizes):
        for depth, node in enumerate(plain_tree.accept(t.parents[b], tokens[b], sampled[b])[0]):
            (p, i), (sp, si) = t.place(b, c + depth), t.place(b, c + node)
            want[:, p, :, i] = t.k[:, sp, :, si]
            moved += node > depth
    assert moved
    path = torch.zeros((2, max(n for _, n in sizes)), dtype=torch.int32, device=DEV)
    flat = lambda x: i32([y for s in x for y in s])
    kernels.tree_accept(flat(tokens), flat(t.parents), d["visible"], flat(sampled), d["cu_q"], 2, path, i32([0, 0]), i32([0, 0]), seq_slot=d["seq_slot"],
                        kv_len=d["kv_len"], block_table=d["block_table"], k=both, v=both)
    assert torch.equal(both.cpu(), want)
