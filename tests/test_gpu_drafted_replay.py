"""A step that checks drafted tokens, captured once and replayed with other trees, paths and rows: bit for bit
what the same calls give eagerly, caches, contexts and what lies past the last token among them."""
import numpy as np
import pytest
import torch

import synth
from gpu_util import from_dev, to_dev
from test_gpu_tree import random_tree

pytestmark = pytest.mark.gpu

ADDED, MOST, ROOM = [9, 4, 20], 24, 40  # nodes, the bound on them, and on all tokens
HEADS, KV, DIM, PAGE, PAGES, HIDDEN, WIDE = 8, 2, 64, 16, 40, 512, 352


class Step:
    def __init__(self, hip, dev, seed):
        rng = np.random.default_rng(seed)
        self.hip, n = hip, len(ADDED)

        def ints(values):
            return to_dev(np.asarray(values, np.int32), dev)

        self.first, self.added = ints(np.cumsum([0, *ADDED])), ints(ADDED)
        self.context, self.length, self.count = ints([30, 0, 101]), ints([0] * n), ints([0] * n)
        self.table = ints(rng.permutation(PAGES)[:n * 13].reshape(n, 13))
        self.parents, self.path = ints([-1] * ROOM), ints(np.zeros((n, MOST)))
        self.slots = torch.full((ROOM,), -1, dtype=torch.int64, device=dev)
        self.cache = torch.zeros(PAGES, hip.kv_q4_0_page_bytes(PAGE, KV, DIM), dtype=torch.uint8, device=dev)
        self.q, self.k, self.v = (torch.zeros(ROOM, h, DIM, device=dev) for h in (HEADS, KV, KV))
        self.bits = torch.zeros(ROOM, 1, dtype=torch.int64, device=dev)
        self.positions = ints([0] * ROOM)
        self.attended = torch.zeros(ROOM, HIDDEN, device=dev)
        self.residual = torch.zeros(ROOM, HIDDEN, device=dev)
        self.rows = torch.zeros(ROOM, HIDDEN // 32 * 34, dtype=torch.uint8, device=dev)
        self.inner = torch.zeros(ROOM, WIDE // 32 * 34, dtype=torch.uint8, device=dev)
        self.gate, self.up = (to_dev(synth.q4_0_matrix(WIDE, HIDDEN, s, 0.1), dev) for s in (3, 4))
        self.turns = torch.empty(512, DIM, device=dev)
        hip.rope_table(DIM, self.turns, 512)
        self.need = hip.attn_tree_q4_0_workspace_bytes("f32", n, ROOM, MOST, 208, HEADS, KV, DIM)
        self.ws = torch.zeros(max(self.need, 16), dtype=torch.uint8, device=dev)

    def load(self, seed):
        """Another step's inputs, from the contexts as they are."""
        rng = np.random.default_rng(seed)
        context, table = from_dev(self.context), from_dev(self.table)
        slots, parents, at = np.full(ROOM, -1, np.int64), np.full(ROOM, -1, np.int32), 0
        path, count = np.zeros((len(ADDED), MOST), np.int32), []
        for r, n in enumerate(ADDED):
            tree = random_tree(rng, n)
            parents[at:at + n] = tree
            t = context[r] + np.arange(n)
            slots[at:at + n] = table[r, t // PAGE].astype(np.int64) * PAGE + t % PAGE
            node, mine = int(rng.integers(0, n)), []
            while node >= 0:
                mine.insert(0, node)
                node = tree[node]
            path[r, :len(mine)] = mine
            count.append(len(mine))
            at += n
        for to, x in ((self.slots, slots), (self.parents, parents), (self.path, path),
                      (self.count, np.array(count, np.int32))):
            to.copy_(torch.from_numpy(x))
        for to in (self.q, self.k, self.v, self.residual):
            to.copy_(torch.from_numpy(rng.standard_normal(tuple(to.shape)).astype(np.float32)))
        torch.cuda.synchronize()

    def run(self):
        hip, n = self.hip, len(ADDED)
        hip.add_i32(self.context, self.added, self.length, n)
        hip.tree_tables(self.parents, self.first, self.length, n, self.bits, 1, self.positions, ROOM)
        hip.rope("f32", "half", self.q, HEADS * DIM, DIM, self.q, HEADS * DIM, DIM, self.positions, self.turns,
                 512, ROOM, HEADS, DIM, DIM)
        hip.kv_store_q4_0("f32", self.k, KV * DIM, DIM, self.v, KV * DIM, DIM, "half", self.positions,
                          self.turns, 512, DIM, self.slots, self.cache, PAGES, PAGE, ROOM, KV, DIM)
        hip.attn_tree_q4_0("f32", self.q, HEADS * DIM, DIM, self.cache, PAGES, PAGE, self.table, 13, self.first,
                           self.length, self.bits, 1, n, ROOM, MOST, 208, HEADS, KV, DIM, DIM ** -0.5, 0,
                           self.attended, HIDDEN, DIM, self.ws, self.need)
        hip.add_rms_norm("f32", self.attended, HIDDEN, self.residual, HIDDEN, self.residual, HIDDEN, None, 1e-5,
                         None, 0, self.rows, self.rows.shape[1], ROOM, HIDDEN)
        hip.gated_q4_0_q8_0("f32", "silu", HIDDEN, None, 0, self.inner, self.inner.shape[1], self.gate, self.up,
                            self.gate.shape[1], self.rows, self.rows.shape[1], WIDE, ROOM)
        hip.kv_keep_q4_0(self.cache, PAGES, PAGE, self.table, 13, self.first, self.length, self.path, MOST,
                         self.count, n, MOST, KV, DIM)
        hip.add_i32(self.context, self.count, self.context, n)

    def state(self):
        torch.cuda.synchronize()
        return {k: from_dev(getattr(self, k)) for k in (
            "context", "length", "bits", "positions", "q", "cache", "attended", "residual", "rows", "inner")}


def test_replays_are_the_eager_steps(hip, dev):
    eager, replayed = Step(hip, dev, 1), Step(hip, dev, 1)
    side = torch.cuda.Stream()
    for s in (eager, replayed):  # a first step, of both
        s.load(100)
        with torch.cuda.stream(side):
            s.run()
        side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        replayed.run()
    for turn in range(4):
        for s in (eager, replayed):
            s.load(101 + turn)
        eager.run()
        graph.replay()
        want, got = eager.state(), replayed.state()
        for name in want:
            assert np.array_equal(want[name].view(np.uint8), got[name].view(np.uint8)), (turn, name)
        assert (got["positions"][sum(ADDED):] == -1).all() and (got["bits"][sum(ADDED):] == 0).all()
        assert (got["attended"][sum(ADDED):] == 0).all()
    assert got["context"].min() > 4 and np.isfinite(got["attended"]).all()
