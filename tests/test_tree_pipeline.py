"""The barriers of csrc/attention_tree_tc5.cu, played with random and lopsided timing: no role waits for good, and nothing is read or overwritten out of
turn.  (A wait tells a phase from the next by its parity only: a wait for V ahead of the one for the tile's scores took the phase of two tiles before for
its own when V was late.  Played evenly that never came up.)"""
import random

import pytest


class Bar:
    """An mbarrier: ``n`` arrivals complete a phase; a wait for parity p passes while the current phase's parity is not p."""

    def __init__(self, n):
        self.n, self.count, self.phase = n, 0, 0

    def arrive(self):
        self.count += 1
        assert self.count <= self.n
        if self.count == self.n:
            self.count, self.phase = 0, self.phase + 1

    def ready(self, parity):
        return (self.phase & 1) != parity


class Block:
    def __init__(self, seed, pieces, stages, warps=4, v_first=False):
        self.rng = random.Random(seed)
        self.pieces, self.stages, self.warps, self.v_first = pieces, stages, warps, v_first
        one = lambda: [Bar(1) for _ in range(stages)]
        self.k_full, self.k_empty, self.v_full, self.v_empty = one(), one(), one(), one()
        self.q_full, self.q_empty, self.o_done, self.o_final = Bar(1), Bar(1), Bar(1), Bar(1)
        self.o_free, self.checked = Bar(warps), Bar(warps)
        self.s_full, self.p_full = [Bar(1), Bar(1)], [Bar(warps), Bar(warps)]
        # what lies where: the tile (or piece) it belongs to
        self.Q, self.K, self.V = None, [None] * stages, [None] * stages
        self.S, self.P, self.O = [None, None], [[None] * warps, [None] * warps], None
        self.flags = [set(), set(), set()]
        self.copies, self.products = [], []              # in flight; products and commits finish in order
        n = sum(pieces)
        coin = lambda p: [[self.rng.random() < p for _ in range(warps)] for _ in range(n)]
        self.masked, self.grows, self.flagged = [self.rng.random() < 0.4 for _ in range(n)], coin(0.5), coin(0.3)

    def loader(self):
        it = 0
        for piece, n in enumerate(self.pieces):
            for j in range(n):
                st, free = it % self.stages, ((it // self.stages) & 1) ^ 1
                yield self.k_empty[st], free
                self.copies.append(("K", st, it, self.k_full[st]))
                if j == 0:
                    if piece:
                        yield self.q_empty, (piece - 1) & 1
                    self.copies.append(("Q", 0, piece, self.q_full))
                yield self.v_empty[st], free
                self.copies.append(("V", st, it, self.v_full[st]))
                it += 1

    def issuer(self):
        def scores(t, done, last, piece):
            if done >= 0:
                yield self.o_done, done & 1
            yield self.k_full[t % self.stages], (t // self.stages) & 1
            self.products += [("S", t, piece), ("commit", self.k_empty[t % self.stages])]
            if last:
                self.products.append(("commit", self.q_empty))
            self.products.append(("commit", self.s_full[t & 1]))
        it = 0
        for piece, n in enumerate(self.pieces):
            yield self.q_full, piece & 1
            yield from scores(it, it - 1, n == 1, piece)
            for j in range(n):
                if j + 1 < n:
                    yield from scores(it + 1, it - 1, j + 2 == n, piece)
                yield self.p_full[it & 1], (it >> 1) & 1
                yield self.v_full[it % self.stages], (it // self.stages) & 1
                if j == 0 and piece:
                    yield self.o_free, (piece - 1) & 1
                self.products += [("O", it, piece), ("commit", self.v_empty[it % self.stages]), ("commit", self.o_done)]
                if j == n - 1:
                    self.products.append(("commit", self.o_final))
                it += 1

    def softmax(self, w):
        it = checks = 0
        for piece, n in enumerate(self.pieces):
            for j in range(n):
                buf, st = it & 1, it % self.stages
                if not self.v_first:
                    yield self.s_full[buf], (it >> 1) & 1
                if self.masked[it]:
                    yield self.v_full[st], (it // self.stages) & 1
                    assert self.V[st] == it
                    if self.flagged[it][w]:
                        self.flags[checks % 3].add((checks, w))
                    yield None
                    if w == 0:
                        self.flags[(checks + 1) % 3].clear()
                    self.checked.arrive()
                    yield self.checked, checks & 1
                    assert self.flags[checks % 3] == {(checks, x) for x in range(self.warps) if self.flagged[it][x]}
                    checks += 1
                if self.v_first:
                    yield self.s_full[buf], (it >> 1) & 1
                assert self.S[buf] == it
                if j > 0 and self.grows[it][w]:
                    yield self.o_done, (it - 1) & 1
                    assert self.O == (piece, it - 1)
                yield None
                assert self.S[buf] == it
                self.P[buf][w] = it
                self.p_full[buf].arrive()
                it += 1
            yield self.o_final, piece & 1
            assert self.O == (piece, it - 1)
            yield None
            assert self.O == (piece, it - 1)
            self.o_free.arrive()

    def land(self, i):
        kind, st, what, bar = self.copies.pop(i)
        if kind == "Q":
            self.Q = what
        else:
            (self.K if kind == "K" else self.V)[st] = what
        bar.arrive()

    def finish(self):
        op = self.products.pop(0)
        if op[0] == "commit":
            op[1].arrive()
        elif op[0] == "S":
            assert self.Q == op[2] and self.K[op[1] % self.stages] == op[1]
            self.S[op[1] & 1] = op[1]
        else:
            t = op[1]
            assert self.V[t % self.stages] == t and self.S[t & 1] == t and all(p == t for p in self.P[t & 1])
            self.O = (op[2], t)

    def play(self):
        roles = [self.loader(), self.issuer()] + [self.softmax(w) for w in range(self.warps)]
        waits, alive = [None] * len(roles), set(range(len(roles)))
        weight = {k: self.rng.choice([1, 1, 0.01, 20]) for k in ("role", "copy", "product")}
        late_v = self.rng.choice([1, 0.005, 30])
        while alive or self.copies or self.products:
            acts = [("role", i, 1) for i in sorted(alive) if waits[i] is None or waits[i][0].ready(waits[i][1])]
            acts += [("copy", i, late_v if c[0] == "V" else 1) for i, c in enumerate(self.copies)]
            if self.products:
                acts.append(("product", 0, 1))
            assert acts, "every role waits"
            kind, i, _ = self.rng.choices(acts, [weight[k] * f for k, _, f in acts])[0]
            if kind == "copy":
                self.land(i)
            elif kind == "product":
                self.finish()
            else:
                try:
                    waits[i] = next(roles[i])
                except StopIteration:
                    alive.discard(i)


def shapes(seed):
    rng = random.Random(seed)
    return [rng.choice([1, 1, 2, 3, rng.randrange(1, 9)]) for _ in range(rng.randrange(1, 6))], rng.choice([2, 4])


@pytest.mark.parametrize("block", range(20))
def test_no_role_waits_for_good_and_nothing_is_out_of_turn(block):
    for seed in range(block * 40, block * 40 + 40):
        Block(seed, *shapes(seed)).play()


def test_a_wait_for_v_ahead_of_the_scores_is_found():
    with pytest.raises(AssertionError):
        for seed in range(400):
            Block(seed, *shapes(seed), v_first=True).play()
