"""Plain forms, in 64 bits on the host, of attention over trees of drafted tokens, of settling such trees and of scoring tokens."""
import math
import random

import torch

PAGE = 64


def bits_of(parents, words):
    """int32 [n, words]: every node's ancestors and itself."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((1 << i) | (rows[p] if p >= 0 else 0))
    return as_words(rows, words)


def as_words(rows, words):
    out = torch.zeros((len(rows), words), dtype=torch.int64)
    for i, r in enumerate(rows):
        for w in range(words):
            out[i, w] = (r >> (32 * w)) & 0xFFFFFFFF
    return torch.where(out >= 2 ** 31, out - 2 ** 32, out).to(torch.int32)


def bit(visible, t, j):
    return (int(visible[t, j // 32]) >> (j % 32)) & 1


def random_parents(rng, n, reach=5):
    return [-1] + [rng.randrange(max(0, i - reach), i) for i in range(1, n)]


class Trees:
    """Sequences of (context, nodes) with pages handed out in no order, on the host."""

    def __init__(self, seed, sizes, nq, nkv, hd, dtype, layers=1, words=None, spare_slots=2):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.sizes, self.nq, self.nkv, self.hd = list(sizes), nq, nkv, hd
        B, most = len(sizes), max([n for _, n in sizes] + [1])
        self.words = words or -(-most // 32)
        pages = [-(-(c + n) // PAGE) for c, n in sizes]
        order = list(range(sum(pages) + 2))
        rng.shuffle(order)
        self.table = torch.full((B + spare_slots, max(pages + [1]) + 1), -1, dtype=torch.int32)
        self.slots = rng.sample(range(B + spare_slots), B)
        for s, p in zip(self.slots, pages):
            for j in range(p):
                self.table[s, j] = order.pop()
        self.unused = order
        n_pages = sum(pages) + 2
        shape = (layers, n_pages, nkv, PAGE, hd)
        self.k, self.v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        self.cu = [0]
        for _, n in sizes:
            self.cu.append(self.cu[-1] + n)
        T = self.cu[-1]
        self.q = (torch.randn((T, nq * hd), generator=g) * 2).to(dtype)
        self.parents = [random_parents(rng, n) for _, n in sizes]
        self.visible = torch.cat([bits_of(p, self.words) for p in self.parents if p] or [torch.zeros((0, self.words), dtype=torch.int32)])[:T]
        self.positions = torch.tensor([c + sum(bit(self.visible, self.cu[b] + i, j) for j in range(n)) - 1
                                       for b, (c, n) in enumerate(sizes) for i in range(n)], dtype=torch.int32)

    def place(self, b, p):
        return int(self.table[self.slots[b], p // PAGE]), p % PAGE

    def ints(self, device):
        i32 = torch.int32
        return dict(block_table=self.table.to(device), seq_slot=torch.tensor(self.slots, dtype=i32, device=device),
                    cu_q=torch.tensor(self.cu, dtype=i32, device=device),
                    kv_len=torch.tensor([c + n for c, n in self.sizes], dtype=i32, device=device), visible=self.visible.to(device))


def attention(t, scale, window=0, keep=0, sinks=None, softcap=0.0, layer=0):
    """float64 [T, nq * hd] and, for every (row, head), sum of weight times |value|: what a rounding of the weights is relative to."""
    group = t.nq // t.nkv
    out = torch.zeros((t.cu[-1], t.nq, t.hd), dtype=torch.float64)
    mass = torch.zeros_like(out)
    for b, (c, n) in enumerate(t.sizes):
        pages = [int(p) for p in t.table[t.slots[b], :-(-(c + n) // PAGE)]]
        k, v = (x[layer, pages].permute(1, 0, 2, 3).reshape(t.nkv, -1, t.hd)[:, :c + n].double() for x in (t.k, t.v))
        for i in range(n):
            row = t.cu[b] + i
            see = [p for p in range(c) if not window or p > int(t.positions[row]) - window or p < keep]
            see += [c + j for j in range(n) if bit(t.visible, row, j)]
            for h in range(t.nq):
                s = k[h // group, see] @ t.q[row, h * t.hd:(h + 1) * t.hd].double() * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if sinks is not None:
                    s = torch.cat([s, sinks[h].double().reshape(1)])
                if not len(s):
                    continue
                w = torch.softmax(s, 0)[:len(see)]
                out[row, h] = w @ v[h // group, see]
                mass[row, h] = w @ v[h // group, see].abs()
    return out.reshape(t.cu[-1], -1), mass.reshape(t.cu[-1], -1)


def accept(parents, tokens, sampled):
    """(path, the token sampled at its end) of one tree."""
    path = [0]
    while True:
        drawn = sampled[path[-1]]
        nxt = next((j for j, up in enumerate(parents) if up == path[-1] and tokens[j] == drawn), None)
        if nxt is None:
            return path, drawn
        path.append(nxt)


def logprobs(x, ids, top):
    """(log probabilities of ids [n, m], entropy [n], the `top` largest and where they are), float64."""
    x = x.double()
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    nothing = torch.isneginf(x).all(1)
    logp[nothing] = -math.inf
    ok = (ids >= 0) & (ids < x.shape[1])
    given = torch.where(ok, logp.gather(1, ids.long().clamp(0, x.shape[1] - 1)), -math.inf)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    value, place = torch.sort(x, dim=1, descending=True, stable=True)
    return given, entropy, logp.gather(1, place[:, :top]), place[:, :top].int()
