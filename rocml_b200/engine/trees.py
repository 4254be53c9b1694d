"""Steps whose sequences bring trees of drafted tokens.

A tree's first node is the token that follows the sequence; every other node is a guess at what follows its parent.  One step runs all of
them: their keys and values go behind the context in the order of the nodes, each node stands at the position that its depth gives it
and sees the context and its ancestors.  ``verify`` then samples at every node, and one kernel finds the path that the samples confirm and moves its keys
and values to the places where ordinary steps would have left them; the pages behind it are given back.

The tokens are those of ordinary generation (but for near ties, which other kernels may round the other way): a sequence's nodes of one
depth share one draw, the one that the step of that token would have used, and the sequence's random stream moves on by as many draws as
tokens were taken.
"""
from __future__ import annotations

import copy
import weakref
from dataclasses import dataclass
from typing import List, Optional, Sequence

import numpy as np
import torch

from .. import kernels
from ..errors import CacheError, ConfigError, RocmlError
from ..profile import profiler as _profiler
from .batch import TREE_WORDS, BatchBuffers, HostBatch, pack_entries

MAX_NODES = kernels.TREE_MAX_NODES


@dataclass
class TreeEntry:
    """``tokens[0]`` follows the sequence of ``slot``; ``parents[i]`` < i is the node that node i follows (-1 for node 0)."""

    slot: int
    tokens: Sequence[int]
    parents: Sequence[int]


def check_tree(entry: TreeEntry, vocab: int) -> None:
    n = len(entry.tokens)
    if not 1 <= n <= MAX_NODES or len(entry.parents) != n:
        raise RocmlError(f"slot {entry.slot}: a tree has 1 to {MAX_NODES} nodes and a parent for each, found {n} and {len(entry.parents)}")
    if entry.parents[0] != -1 or any(not 0 <= p < i for i, p in enumerate(entry.parents) if i):
        raise RocmlError(f"slot {entry.slot}: node 0 has parent -1, every other node an earlier one")
    bad = [t for t in entry.tokens if not 0 <= int(t) < vocab]
    if bad:
        raise RocmlError(f"slot {entry.slot}: token id {bad[0]} is outside the vocabulary of {vocab}")


def pack_trees(old_lens: Sequence[int], parent_lists: Sequence[Sequence[int]]):
    """(positions, parents, rows of bits [T, TREE_WORDS], depths) of a step's trees, node after node."""
    positions, flat, rows, depths = [], [], [], []
    for old, parents in zip(old_lens, parent_lists):
        bits, depth = [], []
        for i, p in enumerate(parents):
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
            depth.append(depth[p] + 1 if p >= 0 else 0)
        positions += [old + d for d in depth]
        flat += [int(p) for p in parents]
        rows += [b.to_bytes(4 * TREE_WORDS, "little") for b in bits]
        depths += depth
    return positions, flat, np.frombuffer(b"".join(rows), dtype="<i4").reshape(len(rows), TREE_WORDS), depths


class _Drawn:
    """A random stream whose next number is known already."""

    def __init__(self, u: float):
        self.u = u

    def next_f32(self) -> float:
        return self.u


class TreeSteps:
    def __init__(self, engine):
        if not engine.model.takes_trees:
            raise ConfigError("this model keeps more than keys and values a sequence, or masks that have no form for trees of drafted tokens")
        # (not a reference that keeps it: an engine that is no longer held gives its memory and its graphs back at once)
        self.engine = weakref.proxy(engine)
        # (a step's logits, one row a node, stay within the head room of the engine's memory budget)
        self.max_nodes = min(engine.max_step_tokens, max(2 * MAX_NODES, engine.cache.max_slots))
        # A node sees all its ancestors: they must lie in every layer's window (its own, whatever the cache keeps for another layer that reads it).
        own = [b.mixer.cache_requirement() for b in engine.model.blocks]
        self.max_depth = min([MAX_NODES] + [int(r.window) for r in own if getattr(r, "window", None)])
        self._buffers = {}
        self._sampler = None

    def _check(self, entries) -> List[TreeEntry]:
        entries = [e if isinstance(e, TreeEntry) else TreeEntry(*e) for e in entries]
        seen = set()
        for e in entries:
            if e.slot in seen:
                raise CacheError(f"slot {e.slot} appears twice in one step")
            seen.add(e.slot)
            check_tree(e, self.engine.model.vocab)
            if len(e.tokens) > self.max_nodes:
                raise RocmlError(f"slot {e.slot}: a tree of {len(e.tokens)} nodes; a step holds {self.max_nodes}")
            depth = max(pack_trees([0], [e.parents])[0]) + 1
            if depth > self.max_depth:
                raise RocmlError(f"slot {e.slot}: a tree {depth} nodes deep; a layer's window holds {self.max_depth} positions")
        # room for everything, before anything launches (every tree beside all others, as if none gave a page back)
        self.engine.cache.plan([[(e.slot, len(e.tokens)) for e in entries]])
        return entries

    def _pieces(self, entries):
        cur, n = [], 0
        for e in entries:
            if cur and (n + len(e.tokens) > self.max_nodes or len(cur) == kernels.TREE_MAX_SEQS):
                yield cur
                cur, n = [], 0
            cur.append(e)
            n += len(e.tokens)
        if cur:
            yield cur

    def _run(self, entries):
        """(logits of a piece's nodes, its buffers on the device, the nodes' depths)."""
        from .engine import _bucket
        eng = self.engine
        slots, tokens = [e.slot for e in entries], [list(e.tokens) for e in entries]
        olds = [eng.cache.grow(e.slot, len(e.tokens)) for e in entries]
        packed = pack_entries(slots, olds, tokens, [range(len(t)) for t in tokens])
        *tree, depths = pack_trees(olds, [e.parents for e in entries])
        T, B, kv_len = len(packed[0]), len(slots), packed[4]
        q_lens = [len(t) for t in tokens]
        host = HostBatch(slots, q_lens, list(kv_len), list(packed[5]))
        eng.cache.flush()
        eng.launches += 1
        eng._device_tokens = None
        eng._replayed = False
        prof = _profiler.ACTIVE
        pads = None
        # short steps are replayed from graphs where short prompts are, if their sizes come back and there is memory for them
        if prof is None and T <= eng._prompt_graph_tokens and eng._tree_sizes.kept:
            t_pad = _bucket(T, 16)
            pads = (t_pad, _bucket(B), t_pad, min(MAX_NODES, _bucket(max(q_lens), 16)), _bucket(max(kv_len), 1024), False)
            due = eng._tree_sizes.due(pads, eng._tree_graphs)
            eng._tree_sizes.note(pads)
            if due:
                logits = eng._run_graph(eng._tree_graphs, eng._tree_sizes.kept, pads, packed, host, T, pads, tree=tree)
                return logits, eng._last_buffers, depths
        key = (_bucket(T, 64), _bucket(B, 8))
        if key not in self._buffers:
            self._buffers[key] = BatchBuffers(key[0], key[1], key[0], eng.device, trees=True)
        buf = self._buffers[key]
        # (padded as the graph will be: an answer does not depend on how often its size has come)
        t_pad, b_pad, w_pad, max_q, max_kv, _ = pads or (T, B, T, max(q_lens), max(kv_len), False)
        buf.fill(*packed, slots, pad_tokens=t_pad, pad_seqs=b_pad, pad_want=w_pad, tree=tree)
        eng.last_h2d_bytes = buf.h2d_bytes
        batch = eng._batch(buf, t_pad, b_pad, w_pad, max_q, max_kv, False, host)
        if prof is None:
            return eng.model.forward(batch, eng.cache)[:T], buf, depths
        with prof.step("prefill", q_lens, kv_len):
            return eng.model.forward(batch, eng.cache), buf, depths

    def logits(self, entries) -> Optional[torch.Tensor]:
        """See ``Engine.tree_logits``."""
        entries = self._check(entries)
        if not entries:
            return None
        pieces = list(self._pieces(entries))
        outs = []
        with torch.cuda.device(self.engine.device):
            for piece in pieces:
                try:
                    got = self._run(piece)[0]
                    outs.append(got.clone() if self.engine._replayed and len(pieces) > 1 else got)
                finally:
                    for e in piece:
                        self.engine.cache.trim(e.slot)
            return outs[0] if len(outs) == 1 else torch.cat(outs, dim=0)

    def verify(self, entries, params, rngs=None, histories=None) -> List[List[int]]:
        """See ``Engine.verify``."""
        entries = self._check(entries)
        n = len(entries)
        rngs = [None] * n if rngs is None else list(rngs)
        histories = [[]] * n if histories is None else list(histories)
        if len(params) != n or len(rngs) != n or len(histories) != n:
            raise RocmlError("verify: parameters, random streams and histories come one an entry")
        for e, p, r in zip(entries, params, rngs):
            if not p.is_greedy and r is None:
                raise RocmlError(f"slot {e.slot}: sampling needs a random stream")
        with torch.cuda.device(self.engine.device):
            try:
                # Everything that can fail comes before any sequence grows or stream moves on: a path's keys and values are moved to places behind its
                # sequence's length, where nothing reads them yet.
                settled, at = [], 0
                for piece in self._pieces(entries):
                    k = len(piece)
                    settled += self._settle_piece(piece, params[at:at + k], rngs[at:at + k], histories[at:at + k])
                    at += k
                results = []
                for e, p, r, (way, last) in zip(entries, params, rngs, settled):
                    self.engine.cache.commit(e.slot, len(way))
                    if not p.is_greedy:
                        for _ in way:
                            r.next_f32()
                    results.append([int(e.tokens[i]) for i in way[1:]] + [last])
                return results
            finally:
                for e in entries:
                    self.engine.cache.trim(e.slot)

    def _settle_piece(self, entries, params, rngs, histories):
        """The confirmed path of every tree, and the token sampled at its end."""
        eng = self.engine
        logits, buf, depths = self._run(entries)
        if self._sampler is None:
            from ..sampling import Sampler
            self._sampler = Sampler(eng.device, max_batch=self.max_nodes)
        row_params, row_rngs, row_histories, row = [], [], [], 0
        for e, p, r, h in zip(entries, params, rngs, histories):
            m = len(e.tokens)
            depth = depths[row:row + m]
            ahead = copy.copy(r) if not p.is_greedy else None       # the stream itself moves on once it is known by how much
            draws = [_Drawn(ahead.next_f32()) for _ in range(max(depth) + 1)] if ahead is not None else None
            row_params += [p] * m
            row_rngs += [None] * m if draws is None else [draws[d] for d in depth]
            if p.repeat_penalty is None:
                row_histories += [h] * m
            else:
                paths = [list(h)]
                for i in range(1, m):
                    paths.append(paths[e.parents[i]] + [int(e.tokens[i])])
                row_histories += paths
            row += m
        handle = self._sampler.launch(logits, row_params, row_rngs, row_histories, status=kernels.status_word(eng.device))
        B, most = len(entries), max(len(e.tokens) for e in entries)
        out = torch.empty(B * (most + 2), dtype=torch.int32, device=eng.device)
        path, counts, nxt = out[:B * most].view(B, most), out[B * most:B * (most + 1)], out[B * (most + 1):]
        tree = buf.tree(row, most)
        settle = lambda **cache: kernels.tree_accept(buf.token_ids, tree.parents, tree.visible, handle.device_tokens, buf.cu_q, B, path, counts,
                                                     nxt, **cache)
        if not eng.cache.kv_groups:
            settle()
        for g in eng.cache.kv_groups:
            settle(seq_slot=buf.seq_slot, kv_len=buf.kv_len, block_table=g.table, k=g.k, v=g.v)
        got = out.cpu()                                  # (this waits for the step)
        kernels.raise_for_status(int(handle.host_status[0]))
        paths, counts, nxt = got[:B * most].view(B, most).tolist(), got[B * most:B * (most + 1)].tolist(), got[B * (most + 1):].tolist()
        return [(way[:count], last) for way, count, last in zip(paths, counts, nxt)]
