"""Trees of drafted tokens without a GPU: how pages are shared among blocks, which words of bits are read, refusals."""
import random

import pytest
import torch

from plain_tree import accept, bits_of, random_parents
from rocml_b200 import kernels
from rocml_b200.errors import KernelError


def pieces_of(sizes, n_shares):
    """What csrc/attention_tree.cu's blocks do with sequences of so many (tiles of keys, tiles of rows): {share: [(sequence, tile of rows, first, end)]}."""
    extra = min(4, sum(t * u for t, u in sizes) // (3 * n_shares))
    pre = [0]
    for t, u in sizes:
        pre.append(pre[-1] + ((t + extra) * u if t else 0))
    out, shares = {}, max(1, min(n_shares, pre[-1]))
    for c in range(shares):
        f, end = c * pre[-1] // shares, (c + 1) * pre[-1] // shares
        b, got = sequence_of(pre, f), []
        while f < end:
            while pre[b + 1] <= f:
                b += 1
            mt, p0 = divmod(f - pre[b], sizes[b][0] + extra)
            stop = min(sizes[b][0] + extra, p0 + end - f)
            f += stop - p0
            if p0 < sizes[b][0]:
                got.append((b, mt, p0, min(stop, sizes[b][0])))
        out[c] = got
    return pre, out, shares, extra


def sequence_of(pre, f):
    lo, hi = 0, len(pre) - 2
    while lo < hi:
        mid = (lo + hi + 1) >> 1
        lo, hi = (mid, hi) if pre[mid] <= f else (lo, mid - 1)
    return lo


@pytest.mark.parametrize("seed", range(60))
def test_shares_cover_every_tile_once_and_pieces_have_places_of_their_own(seed):
    rng = random.Random(seed)
    sizes = [(t, rng.choice([1, 1, 2, 5]) if t else 0) for t in [rng.choice([0, 1, 2, 3, rng.randrange(1, 200)]) for _ in range(rng.randrange(1, 40))]]
    shares = rng.choice([1, 2, 3, 17, 18, 37, 296])
    pre, pieces, shares, extra = pieces_of(sizes, shares)
    W = pre[-1]
    seen, places = {}, {}
    for c, got in pieces.items():
        for b, mt, p0, p1 in got:
            assert 0 <= p0 < p1 <= sizes[b][0] and 0 <= mt < sizes[b][1]
            seen.setdefault((b, mt), []).extend(range(p0, p1))
            if not (p0 == 0 and p1 == sizes[b][0]):
                place = 2 * c + (1 if p0 == 0 else 0)
                assert place < 2 * shares and place not in places        # nobody else's, inside the work space
                places[place] = (b, mt)
    for b, (t, u) in enumerate(sizes):
        for mt in range(u):
            assert sorted(seen.pop((b, mt))) == list(range(t))
    assert not seen
    # the notes that the joining kernel reads: one a (sequence, tile of rows), or one a share
    share_of = lambda g: ((g + 1) * shares - 1) // W
    by_unit, by_share, joined = {}, {}, {}
    for c, got in pieces.items():
        f, end = c * W // shares, (c + 1) * W // shares
        for b, mt, p0, p1 in got:
            if p0 == 0:
                last = c if p1 == sizes[b][0] else share_of(pre[b] + mt * (sizes[b][0] + extra) + sizes[b][0] - 1)
                assert (b, mt) not in by_unit
                by_unit[b, mt] = (c, last)
                if last != c:
                    assert c not in by_share
                    by_share[c] = (b, mt, last)
        cuts = False
        if c + 1 < shares and f < end:
            b = sequence_of(pre, end)
            into = (end - pre[b]) % (sizes[b][0] + extra)
            cuts = 0 < into < sizes[b][0] and end - into >= f
        assert cuts == (c in by_share)
    for (b, mt), (c0, c1) in by_unit.items():
        for c in range(c0, c1 + 1) if c0 != c1 else ():
            joined[2 * c + (1 if c == c0 else 0)] = (b, mt)
    assert joined == places and sorted(by_unit) == [(b, mt) for b, (_, u) in enumerate(sizes) for mt in range(u)]
    assert {(b, mt): (c, last) for c, (b, mt, last) in by_share.items()} == {k: v for k, v in by_unit.items() if v[0] != v[1]}


@pytest.mark.parametrize("off", [-63, -64, -33, -32, -31, -1, 0, 1, 31, 32, 63, 64, 200, 255])
def test_a_tiles_words_of_bits(off):
    """The funnel of three words that csrc/attention_tree.cu builds a tile's 64 bits from."""
    rng = random.Random(off)
    n = 256
    row = rng.getrandbits(n)
    words = [(row >> (32 * w)) & 0xFFFFFFFF for w in range(8)]
    w0, sh = off >> 5, off & 31
    w = [words[w0 + i] if 0 <= w0 + i < 8 else 0 for i in range(3)]
    lo = ((w[1] << 32 | w[0]) >> sh) & 0xFFFFFFFF
    hi = ((w[2] << 32 | w[1]) >> sh) & 0xFFFFFFFF
    want = sum(((row >> j) & 1) << (j - off) for j in range(max(0, off), min(n, off + 64)))
    mask = sum(1 << i for i in range(64) if 0 <= off + i < n)
    assert ((hi << 32) | lo) & mask == want


@pytest.mark.parametrize("seed", range(30))
def test_confirmed_nodes_by_bits_are_the_walk(seed):
    """(visible & ~like) == 0 names the nodes that a walk from node to node reaches, and their depth is their place."""
    rng = random.Random(seed)
    n = rng.randrange(1, 70)
    parents = random_parents(rng, n, rng.choice([1, 2, 9]))
    tokens, sampled = [rng.randrange(3) for _ in range(n)], [rng.randrange(3) for _ in range(n)]
    path, drawn = accept(parents, tokens, sampled)
    rows = bits_of(parents, 3)
    first = {}
    for i in range(1, n):
        if tokens[i] == sampled[parents[i]]:
            first.setdefault(parents[i], i)
    like = sum(1 << i for i in range(n) if i == 0 or first.get(parents[i]) == i)
    whole = [sum((int(rows[i, w]) & 0xFFFFFFFF) << (32 * w) for w in range(3)) for i in range(n)]
    kept = [i for i in range(n) if whole[i] & ~like == 0]
    assert sorted(kept, key=lambda i: bin(whole[i]).count("1")) == path
    assert [bin(whole[i]).count("1") - 1 for i in path] == list(range(len(path)))
    assert drawn == sampled[path[-1]]


def test_shares_fill_the_device_and_never_outnumber_the_pages():
    assert kernels.tree_shares(200, 1, 64, 8, 296) == 37
    assert kernels.tree_shares(200, 1, 128, 8, 296) == 25
    assert kernels.tree_shares(14, 14, 128, 8, 296) == 14
    assert kernels.tree_shares(324, 36, 26, 8, 296) == 36 and kernels.tree_shares(324, 20, 26, 8, 296) == 37
    assert kernels.tree_shares(3, 1, 16, 8, 296) == 3
    assert kernels.tree_shares(320, 32, 5, 1000, 296) == 2
    assert kernels.tree_shares(1, 1, 128, 5000, 296) == 1


def test_clusters_stay_small_and_together_on_the_device():
    for n_pages in (1, 2, 3, 8, 16, 17, 40, 41, 72, 73, 144, 145, 2000):
        for units in (1, 2, 3, 8, 37, 1000):
            for rows in (1, 16, 32, 33, 64, 128):
                for nkv in (1, 3, 8, 16, 200):
                    for slots in (148, 296):
                        c = kernels.tree_cluster(n_pages, units, rows, nkv, slots)
                        assert 0 <= c <= 16 and c != 1
                        if c:
                            assert units * nkv * c <= slots and n_pages <= 9 * c and c <= n_pages
                            assert c <= 8 or (rows <= 32 and 2 * units * nkv * c <= slots)
    assert [kernels.tree_cluster(p, 1, 16, 8, 296) for p in (1, 2, 5, 16, 17, 144, 145)] == [0, 2, 5, 7, 16, 16, 0]
    assert [kernels.tree_cluster(p, 1, 128, 8, 296) for p in (5, 35, 36)] == [5, 7, 0]
    assert [kernels.tree_cluster(16, b, 64, 8, 296) for b in (1, 4, 6, 8, 16, 17)] == [7, 7, 5, 4, 0, 0]


def _attention(**change):
    """A call that is right but for living on the host."""
    i32 = torch.int32
    a = dict(q=torch.zeros((5, 8 * 64)), out=torch.zeros((5, 8 * 64)), k_cache=torch.zeros((3, 2, 64, 64)), v_cache=torch.zeros((3, 2, 64, 64)),
             block_table=torch.zeros((2, 3), dtype=i32), seq_slot=torch.zeros(2, dtype=i32), cu_q=torch.zeros(3, dtype=i32),
             kv_len=torch.zeros(2, dtype=i32), visible=torch.zeros((5, 1), dtype=i32), n_seqs=2, max_nodes=4, nq=8, nkv=2, hd=64, scale=0.1)
    a.update(change)
    kernels.attention_tree(**a)


@pytest.mark.parametrize("change, says", [
    ({}, "there is no CPU path"),
    ({"max_nodes": 33}, "33 nodes in 1 words"),
    ({"visible": torch.zeros((5, 9), dtype=torch.int32)}, "9 words"),
    ({"visible": torch.zeros((5, 1), dtype=torch.int64)}, "int32"),
    ({"visible": torch.zeros((6, 1), dtype=torch.int32)}, "a row of nq"),
    ({"n_seqs": 3}, "3 sequences"),
    ({"nq": 7}, "cache must be"),
    ({"hd": 32}, "cache must be"),
    ({"q": torch.zeros((5, 512), dtype=torch.bfloat16)}, "one type"),
    ({"scale": 0.0}, "scale is positive"),
    ({"window": 5}, "positions"),
    ({"window": -5}, "not negative"),
    ({"v_cache": torch.zeros((3, 2, 64, 128))[..., :64]}, "contiguous"),
])
def test_attention_tree_refuses(change, says):
    with pytest.raises(KernelError, match=says):
        _attention(**change)


def _accept(**change):
    i32 = torch.int32
    a = dict(token_ids=torch.zeros(5, dtype=i32), parents=torch.zeros(5, dtype=i32), visible=torch.zeros((5, 1), dtype=i32),
             sampled=torch.zeros(5, dtype=i32), cu_q=torch.zeros(3, dtype=i32), n_seqs=2, path=torch.zeros((2, 4), dtype=i32),
             counts=torch.zeros(2, dtype=i32), next_token=torch.zeros(2, dtype=i32))
    a.update(change)
    kernels.tree_accept(**a)


@pytest.mark.parametrize("change, says", [
    ({}, "there is no CPU path"),
    ({"parents": torch.zeros(4, dtype=torch.int32)}, "for every node"),
    ({"counts": torch.zeros(1, dtype=torch.int32)}, "for every sequence"),
    ({"path": torch.zeros((2, 300), dtype=torch.int32)}, "at most 256"),
    ({"path": torch.zeros((1, 4), dtype=torch.int32)}, "n_seqs"),
    ({"v": torch.zeros((1, 2, 1, 64, 16))}, "come with keys"),
    ({"k": torch.zeros((1, 2, 1, 64, 16)), "v": torch.zeros((1, 2, 1, 64, 16))}, "needs seq_slot"),
])
def test_tree_accept_refuses(change, says):
    with pytest.raises(KernelError, match=says):
        _accept(**change)


@pytest.mark.parametrize("change, says", [
    ({}, "there is no CPU path"),
    ({"ids": None}, "come together"),
    ({"top_ids": torch.zeros((3, 33), dtype=torch.int32), "top_logprobs": torch.zeros((3, 33))}, "at most 32"),
    ({"logits": torch.zeros((50, 3)).t()}, "unit inner stride"),
    ({"entropy": torch.zeros(2)}, "entropy"),
    ({"logprobs": torch.zeros((3, 2), dtype=torch.float64)}, "contiguous float32"),
])
def test_token_logprobs_refuses(change, says):
    a = dict(logits=torch.zeros((3, 50)), ids=torch.zeros((3, 2), dtype=torch.int32), logprobs=torch.zeros((3, 2)))
    a.update(change)
    with pytest.raises(KernelError, match=says):
        kernels.token_logprobs(**a)
