"""Drafted tokens as trees over the paged Q4_0 cache on the GPU: tables and moved rows exactly, attention
against float64 with the tolerances of test_gpu_kv_cache.Setup."""
import numpy as np
import pytest
import torch

import kv_plain
from gpu_util import from_dev, to_dev
from test_gpu_kv_cache import ELEMS, TORCH, Setup, dev_rows, wide

pytestmark = pytest.mark.gpu


def random_tree(rng, nodes, chain=0.5):
    return [int(j - 1 if rng.random() < chain else rng.integers(-1, j)) for j in range(nodes)]


def bits_of(tree):
    """[nodes][nodes] truth values: a node and its ancestors; and the depths."""
    seen, depth = np.zeros((len(tree), len(tree)), bool), []
    for j, p in enumerate(tree):
        up = p if -1 < p < j else -1
        if up >= 0:
            seen[j] = seen[up]
        seen[j, j] = True
        depth.append(depth[up] + 1 if up >= 0 else 0)
    return seen, depth


def words_of(trees, words):
    rows = np.zeros((sum(len(t) for t in trees), words), np.uint64)
    at = 0
    for tree in trees:
        seen = bits_of(tree)[0]
        for j in range(len(tree)):
            for i in np.flatnonzero(seen[j]):
                if i < 64 * words:
                    rows[at + j, i // 64] |= np.uint64(1) << np.uint64(i % 64)
        at += len(tree)
    return rows


# ---------------------------------------------------------------- tables ---

@pytest.mark.parametrize("nodes,words,room", [
    ([1], 1, 0), ([64], 1, 3), ([65], 2, 0), ([0, 5, 0, 0, 9], 1, 1), ([300, 1, 17], 5, 0),
    ([130, 70], 2, -20), ([200], 2, 0), ([9000], 1, 0), ([3] * 400, 1, 60), ([12, 12], 3, -12),
    ([5, 3], 2, 3000), ([4096, 64, 128], 64, 0), ([4200, 4097], 66, 2), ([4160], 3, 0),
])
def test_tables(hip, dev, nodes, words, room):
    """Also nodes that have no bits, more tokens than are asked for, and parents that are none."""
    rng = np.random.default_rng(sum(nodes) + words)
    trees = [random_tree(rng, n, 0.9 if n < 1000 else 0.5) for n in nodes]
    for tree in trees:
        if len(tree) > 8:
            tree[3], tree[5], tree[7] = 3, 7, -5
    parents = np.array([p for t in trees for p in t] + [0], np.int32)
    first = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    cached = rng.integers(0, 1000, len(nodes))
    length = (cached + nodes).astype(np.int32)
    total, most = int(first[-1]), int(first[-1]) + room
    want = np.zeros((most, words), np.uint64)
    where = np.full(most, -1, np.int32)
    keep = min(total, most)
    want[:keep] = words_of(trees, words)[:keep]
    where[:keep] = np.concatenate([c + np.array(bits_of(t)[1], np.int64).reshape(-1)
                                   for c, t in zip(cached, trees)])[:keep]
    bits = torch.full((most + 1, words), 0x5555, dtype=torch.int64, device=dev)
    positions = torch.full((most + 1,), 99, dtype=torch.int32, device=dev)
    hip.tree_tables(to_dev(parents, dev), to_dev(first, dev), to_dev(length, dev), len(nodes), bits,
                    words, positions, most)
    got = from_dev(bits)
    assert np.array_equal(got[:most].view(np.uint64), want) and (got[most:] == 0x5555).all()
    got = from_dev(positions)
    assert np.array_equal(got[:most], where) and (got[most:] == 99).all()


@pytest.mark.parametrize("nodes", [64, 65, 640, 4300])
def test_tables_of_chains_and_stars(hip, dev, nodes):
    """The deepest tree, the flattest, one whose paths go through every second word, and one by twos."""
    words = -(-nodes // 64)
    i = np.arange(nodes)
    for parents in (i - 1, np.zeros_like(i) - (i == 0), i - 65, i - 2):
        tree = [int(max(p, -1)) for p in parents]
        bits = torch.zeros(nodes, words, dtype=torch.int64, device=dev)
        positions = torch.zeros(nodes, dtype=torch.int32, device=dev)
        hip.tree_tables(to_dev(np.array(tree, np.int32), dev), to_dev(np.array([0, nodes], np.int32), dev),
                        to_dev(np.array([nodes + 7], np.int32), dev), 1, bits, words, positions, nodes)
        assert np.array_equal(from_dev(bits).view(np.uint64), words_of([tree], words))
        assert from_dev(positions).tolist() == [7 + d for d in bits_of(tree)[1]]


def test_tables_of_nothing(hip, dev):
    bits = torch.full((3, 1), 5, dtype=torch.int64, device=dev)
    positions = torch.full((3,), 5, dtype=torch.int32, device=dev)
    hip.tree_tables(None, None, None, 0, bits, 1, positions, 3)
    assert (from_dev(bits) == 0).all() and (from_dev(positions) == -1).all()


# ------------------------------------------------------------- attention ---

class Trees(Setup):
    """Requests whose new tokens are the nodes of trees."""

    def __init__(self, dev, elem, cached, nodes, heads, kv, dim, page, seed=0, chain=0.5, **kw):
        super().__init__(dev, elem, [c + n for c, n in zip(cached, nodes)], nodes, heads, kv, dim,
                         page, seed=seed, **kw)
        rng = np.random.default_rng(seed + 5)
        self.trees = [random_tree(rng, n, chain) for n in nodes]
        self.words = max(1, -(-max(nodes) // 64))
        self.bits = words_of(self.trees, self.words)

    def run(self, hip, window=0, scale=None, out=None, bits=None, max_added=None, max_length=None,
            tokens=None, words=None, bufs=None, stream=None):
        heads, kv, dim, elem = self.heads, self.kv, self.dim, self.elem
        scale = dim ** -0.5 if scale is None else scale
        n, tokens = len(self.lengths), tokens or self.tokens
        q = dev_rows(self.q, elem, self.dev)
        out = torch.full((tokens, heads, dim), 3.0, dtype=TORCH[elem], device=self.dev) \
            if out is None else out
        most_a = int(self.added.max()) if max_added is None else max_added
        most_l = int(self.lengths.max()) if max_length is None else max_length
        need = hip.attn_tree_q4_0_workspace_bytes(elem, n, tokens, most_a, most_l, heads, kv, dim)
        ws = torch.full((max(need // 4, 4),), float("nan"), device=self.dev)
        b = bufs or self.buffers()
        bits = self.bits if bits is None else bits
        hip.attn_tree_q4_0(elem, q, q.stride(0), q.stride(1), b[0], self.pages, self.page, b[1],
                           self.stride, b[2], b[3], to_dev(bits.view(np.int64), self.dev),
                           words or bits.shape[1], n, tokens, most_a, most_l, heads, kv, dim, scale,
                           window, out, out.stride(0), out.stride(1), ws, need, stream)
        return out

    def want(self, scale=None, window=0, bits=None):
        scale = np.float64(np.float32(self.dim ** -0.5 if scale is None else scale))
        bits = self.bits if bits is None else bits
        out = np.zeros((self.tokens, self.heads, self.dim))
        share = self.heads // self.kv
        for r in range(len(self.lengths)):
            length, n = int(self.lengths[r]), int(self.added[r])
            cached = length - n
            for i in range(n):
                row = bits[self.first[r] + i]
                mine = [j for j in range(i + 1) if int(row[j // 64]) >> (j % 64) & 1]
                p = cached + max(len(mine), 1) - 1
                low = max(0, p - window + 1) if window else 0
                seen = list(range(min(low, cached), cached))
                seen += [cached + j for d, j in enumerate(mine) if not window or cached + d >= low]
                if not seen:
                    continue
                for h in range(self.heads):
                    q = self.q[self.first[r] + i, h].astype(np.float64)
                    z = scale * (self.k[r][seen, h // share] @ q)
                    w = np.exp(z - z.max())
                    out[self.first[r] + i, h] = w @ self.v[r][seen, h // share] / w.sum()
        return out

    def check(self, hip, **kw):
        got = wide(self.run(hip, **kw))
        want = self.want(**{k: v for k, v in kw.items() if k in ("scale", "window", "bits")})
        off = np.abs(got - want)
        assert np.isfinite(got).all()
        assert (off <= self.tolerance(want, kw.get("scale"))).all(), off.max()
        return got


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("cached,nodes,heads,kv,dim,page", [
    ([0], [1], 1, 1, 64, 16),
    ([0, 1, 15, 16], [5, 1, 8, 3], 4, 1, 64, 16),
    ([31, 32, 33], [4, 31, 33], 8, 2, 128, 16),
    ([5, 530, 97], [7, 0, 12], 32, 8, 128, 48),
    ([300, 1000], [64, 40], 14, 2, 64, 32),
    ([77, 200], [9, 2], 4, 4, 192, 16),
    ([200, 40], [3, 20], 8, 1, 256, 64),
    ([2100, 40], [6, 6], 8, 2, 64, 16),      # split over work-groups and joined
    ([900, 3], [130, 70], 4, 2, 64, 16),     # three words
    ([4000], [2], 4, 1, 128, 128),
    ([700], [65], 40, 1, 128, 16),
    ([5, 0, 60], [0, 0, 3], 6, 2, 128, 16),
    # tiles of few stretches and of many, rows of heads that one work-group's groups hold side by side or not
    ([700, 1300, 2600, 6000], [3, 1, 4, 2], 4, 1, 256, 16),
    ([700, 1300, 2600, 5000, 90], [3, 9, 4, 2, 12], 4, 1, 64, 16),
    ([400, 900, 1700], [5, 3, 1], 14, 2, 192, 32),
])
def test_trees(hip, dev, elem, cached, nodes, heads, kv, dim, page):
    t = Trees(dev, elem, cached, nodes, heads, kv, dim, page, seed=len(cached))
    t.check(hip)
    for window in (1, 3, 40):
        t.check(hip, window=window)


# (cached, nodes, heads, kv_heads, dim, page) whose windowed rows are shared out and joined; which kernels
# they take is pinned by test_more_dispatch.py
WINDOWED = [
    # several tiles a kv head, in parts: each tile's range begins with what the first node sees
    ([4100, 300, 2500], [200, 70, 130], 8, 2, 64, 16),
    ([3500, 5000], [200, 3], 8, 2, 128, 32),
    ([2900], [330], 4, 2, 192, 16),
    ([3300], [150], 8, 2, 256, 16),
    # up to 64 rows, in stretches
    ([5000, 4100, 90], [16, 9, 16], 8, 2, 128, 16),
    ([6000], [61], 2, 2, 64, 16),
    ([3900, 800], [12, 16], 4, 1, 256, 48),
]


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("cached,nodes,heads,kv,dim,page", WINDOWED)
def test_windows_over_parts(hip, dev, elem, cached, nodes, heads, kv, dim, page):
    """Long windows, whose tiles are in parts: a late node of little depth sees more of the cached tokens
    than its number among the nodes would leave."""
    t = Trees(dev, elem, cached, nodes, heads, kv, dim, page, seed=15)
    for window in (700, 3000):
        t.check(hip, window=window)


@pytest.mark.parametrize("elem", ELEMS)
def test_many_requests(hip, dev, elem):
    rng = np.random.default_rng(2)
    cached = [int(x) for x in rng.integers(0, 900, 70)]
    nodes = [int(x) for x in rng.integers(0, 12, 70)]
    nodes[0] = 12
    t = Trees(dev, elem, cached, nodes, 8, 4, 64, 16, seed=3)
    t.check(hip)
    t.check(hip, window=200, scale=-0.3)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("nodes", [1, 8, 90])
def test_a_chain_is_causal(hip, dev, elem, nodes):
    """Each node the child of the one before: what attn_q4_0 computes, within both's tolerance."""
    t = Trees(dev, elem, [700, 90], [nodes, nodes], 8, 2, 128, 32, seed=6, chain=2.0)
    assert (t.bits[0] == [1] + [0] * (t.words - 1)).all()
    for window in (0, 50):
        got = t.check(hip, window=window)
        other = wide(Setup.run(t, hip, window=window))
        tol = 2 * t.tolerance(Setup.want(t, window=window))
        assert (np.abs(got - other) <= tol).all()


@pytest.mark.parametrize("elem", ELEMS)
def test_rows_without_bits(hip, dev, elem):
    """A row whose bits leave nothing sees the cached tokens alone, and none of them is zero; bits past a
    token's own are not looked at."""
    t = Trees(dev, elem, [0, 40, 3], [6, 6, 70], 4, 2, 64, 16, seed=7)
    bits = t.bits.copy()
    bits[2] = 0
    bits[8] = 0
    bits[15, :] = 0
    for window in (0, 4):
        got = t.check(hip, window=window, bits=bits)
        assert (got[2] == 0).all() and not (got[8] == 0).any()
        more = bits.copy()
        for r in range(3):
            for j in range(int(t.added[r])):
                row = more[t.first[r] + j]
                for i in range(j + 1, 64 * t.words):
                    row[i // 64] |= np.uint64(1) << np.uint64(i % 64)
        assert np.array_equal(wide(t.run(hip, window=window, bits=more)), got)


@pytest.mark.parametrize("elem", ELEMS)
def test_what_a_row_does_not_see(hip, dev, elem):
    """Siblings that hold NaN and infinities, and pages that are missing."""
    t = Trees(dev, elem, [37, 200], [20, 9], 8, 2, 64, 16, seed=8)
    t.trees = [[-1] + [0] * 19, [-1] + list(range(8))]
    t.bits = words_of(t.trees, 1)
    want = t.want()
    clean = wide(t.run(hip))
    for j in range(1, 20):  # all but the root: each of them is seen by itself only
        slot = int(t.table[0, (37 + j) // 16]) * 16 + (37 + j) % 16
        for which in "kv":
            for h in range(t.kv):
                t.cache.put(slot, h, which, np.full(2, [np.nan, np.inf][j % 2], np.float16),
                            np.full((2, 16), 0xFF, np.uint8))
    got = wide(t.run(hip))
    assert np.array_equal(got[0], clean[0]) and np.array_equal(got[20:], clean[20:])
    assert not np.isfinite(got[1:20]).any()
    table = t.table.copy()
    table[1, 2] = -1  # tokens 32 .. 47
    bufs = list(t.buffers())
    bufs[1] = to_dev(table, dev)
    t.k[1], t.v[1] = np.delete(t.k[1], range(32, 48), 0), np.delete(t.v[1], range(32, 48), 0)
    t.lengths[1] -= 16
    got = wide(t.run(hip, bufs=tuple(bufs), max_length=int(t.lengths[1]) + 16))
    want = t.want()
    assert (np.abs(got[20:] - want[20:]) <= t.tolerance(want)[20:] if elem != "f32"
            else np.abs(got[20:] - want[20:]) <= t.tolerance(want)).all()


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("cached,nodes,share", [([-10, 47], [30, 3], 2), ([-80, -1], [130, 5], 4)])
def test_windows_wider_than_all_positions(hip, dev, elem, cached, nodes, share):
    """They hide nothing, also where a request has fewer tokens than nodes, the first of which lie before
    token 0 then and are not there."""
    t = Trees(dev, elem, cached, nodes, 2 * share, 2, 64, 16, seed=14, chain=0.8)
    whole = wide(t.run(hip))
    for window in (2 ** 30, 2 ** 31 - 20, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 32 + 1):
        assert np.array_equal(wide(t.run(hip, window=window)), whole), window
    want = np.zeros_like(whole, dtype=np.float64)
    for r, tree in enumerate(t.trees):
        for i, sees in enumerate(bits_of(tree)[0]):
            seen = list(range(cached[r])) + [cached[r] + j for j in np.flatnonzero(sees)]
            seen = [x for x in seen if x >= 0]
            for h in range(t.heads if seen else 0):
                z = 0.125 * (t.k[r][seen, h // share] @ t.q[t.first[r] + i, h].astype(np.float64))
                w = np.exp(z - z.max())
                want[t.first[r] + i, h] = w @ t.v[r][seen, h // share] / w.sum()
    assert (np.abs(whole - want) <= t.tolerance(want)).all() and (whole != 0).any()


def test_bounds_rows_past_the_last_and_strides(hip, dev):
    t = Trees(dev, "f16", [50, 90], [5, 7], 4, 2, 64, 16, seed=9)
    want = wide(t.run(hip))
    out = torch.full((15, 6, 80), 3.0, dtype=torch.float16, device=dev)
    t.run(hip, out=out, max_added=30, max_length=4096, tokens=15)
    got = wide(out)
    assert (got[12:] == 3.0).all() and (got[:, 4:] == 3.0).all() and (got[:, :, 64:] == 3.0).all()
    assert np.abs(got[:12, :4, :64] - want).max() <= 2.0 ** -9 * np.abs(want).max()
    wider = np.concatenate([t.bits, np.full((12, 2), ~np.uint64(0))], 1)  # words that no node has
    assert np.array_equal(wide(t.run(hip, bits=wider)), want)


def test_same_bits_on_another_stream_and_replayed(hip, dev):
    t = Trees(dev, "f32", [2500, 90], [9, 30], 8, 2, 64, 16, seed=10)
    want = wide(t.run(hip))
    side = torch.cuda.Stream()
    bufs, q = t.buffers(), dev_rows(t.q, "f32", dev)
    bits = to_dev(t.bits.view(np.int64), dev)
    need = hip.attn_tree_q4_0_workspace_bytes("f32", 2, t.tokens, 30, 2509, 8, 2, 64)
    assert need > 0
    ws, out = torch.zeros(need, dtype=torch.uint8, device=dev), torch.zeros_like(q)
    torch.cuda.synchronize()

    def step():
        hip.attn_tree_q4_0("f32", q, 512, 64, bufs[0], t.pages, 16, bufs[1], t.stride, bufs[2],
                           bufs[3], bits, 1, 2, t.tokens, 30, 2509, 8, 2, 64, 0.125, 0, out, 512, 64,
                           ws, need)

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert np.array_equal(wide(out), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(3):
        out.zero_()
        ws.zero_()
        torch.cuda.synchronize()
        graph.replay()
        assert np.array_equal(wide(out), want)


# ------------------------------------------------------------------ keep ---

def kept_plain(t, cached, nodes, paths, max_added=None):
    """The cache's bytes after the path's rows have moved, token by token and all read first."""
    before, after = t.cache.bytes.copy(), t.cache.bytes.copy()
    for r, path in enumerate(paths):
        most = nodes[r] if max_added is None else min(nodes[r], max_added)
        for k, node in enumerate(path[:most]):
            if not 0 <= node < most:
                continue
            a, b = cached[r] + node, cached[r] + k
            pages = [int(t.table[r, x // t.page]) if x // t.page < t.stride else -1 for x in (a, b)]
            if min(pages) < 0 or max(pages) >= t.pages:
                continue
            for old, new in row_places(t, a % t.page, b % t.page):
                after[pages[1], :, new] = before[pages[0], :, old]
    return after


def row_places(t, a, b):
    c, nb = t.cache, t.dim // 32
    base = c.quants + c.scales

    def places(x):
        got = [(x * 4) * nb * 4 + i for i in range(16 * nb)]
        for at in (c.quants, base + c.quants):
            got += [at + ((x // 4) * nb + i) * 8 + (x % 4) * 2 + e for i in range(nb) for e in range(2)]
        return got + [base + (((x // 4) * 16 + m) * (nb // 2) + i) * 8 + (x % 4) * 2 + e
                      for m in range(16) for i in range(nb // 2) for e in range(2)]
    return zip(places(a), places(b))


@pytest.mark.parametrize("dim,kv,page", [(64, 1, 16), (128, 3, 32), (192, 2, 16), (256, 2, 48)])
@pytest.mark.parametrize("cached,nodes", [
    ([0], [1]), ([7, 30, 100], [20, 64, 5]), ([13], [200]), ([0, 15, 16, 17], [9, 0, 40, 3]),
])
def test_keep(hip, dev, dim, kv, page, cached, nodes):
    t = Trees(dev, "f16", cached, nodes, kv, kv, dim, page, seed=11, chain=0.3)
    rng = np.random.default_rng(1)
    paths = []
    for n in nodes:
        size = int(rng.integers(0, n + 1)) if n > 1 else n
        paths.append(sorted(rng.choice(n, size, replace=False).tolist()))
    width = max(nodes) + 1
    path = np.full((len(nodes), width), -7, np.int32)
    for r, p in enumerate(paths):
        path[r, :len(p)] = p
    want = kept_plain(t, cached, nodes, paths)
    b = t.buffers()
    count = to_dev(np.array([len(p) for p in paths], np.int32), dev)
    hip.kv_keep_q4_0(b[0], t.pages, page, b[1], t.stride, b[2], b[3], to_dev(path, dev), width, count,
                     len(nodes), max(nodes), kv, dim)
    got = from_dev(b[0]).reshape(want.shape)
    assert np.array_equal(got, want)


def test_keep_of_what_is_not_there(hip, dev):
    """Nodes that the request has not, counts past the path and the tree, missing pages, fewer nodes
    looked at: the rest moves, and nothing else changes."""
    cached, nodes = [10, 20, 5], [30, 8, 40]
    t = Trees(dev, "f16", cached, nodes, 2, 2, 64, 16, seed=12)
    t.table[2, 1] = -1
    t.table[2, 2] = t.pages
    paths = [[1, 99, -4, 5, 6, 2 ** 31 - 1, 29], [0, 1, 2, 5, 6, 7, 8], [3, 8, 30, 33, 39, 40, 41]]
    path = np.array(paths, np.int32)
    for most in (40, 7):
        want = kept_plain(t, cached, nodes, paths, most)
        b = t.buffers()
        hip.kv_keep_q4_0(b[0], t.pages, 16, b[1], t.stride, b[2], b[3], to_dev(path, dev), 7,
                         to_dev(np.array([100, 2 ** 31 - 1, 7], np.int32), dev), 3, most, 2, 64)
        assert np.array_equal(from_dev(b[0]).reshape(want.shape), want)
    b = t.buffers()
    hip.kv_keep_q4_0(b[0], t.pages, 16, b[1], t.stride, b[2], b[3], to_dev(path, dev), 7,
                     to_dev(np.array([0, -3, -2 ** 31], np.int32), dev), 3, 40, 2, 64)
    assert np.array_equal(from_dev(b[0]).reshape(t.cache.bytes.shape), t.cache.bytes)


# ------------------------------------------------------- caches past 4 GiB ---

@pytest.mark.parametrize("nodes", [[7, 16], [80, 2]])
def test_pages_past_32_bits(hip, dev, nodes):
    """The pages lie more than 2^32 bytes into the cache: the same attention and the same moves."""
    t = Trees(dev, "f16", [300, 90], nodes, 8, 2, 128, 16, seed=13)
    want = wide(t.run(hip))
    near = t.buffers()
    page_bytes = near[0].numel() // t.pages
    pages = (9 << 30) // page_bytes
    cache = torch.empty(pages * page_bytes, dtype=torch.uint8, device=dev)
    base = pages - t.pages
    cache[base * page_bytes:] = near[0].view(-1)
    used = (near[1] >= 0) & (near[1] < t.pages)
    far = [cache, torch.where(used, near[1] + base, near[1].clamp(max=-1)), *near[2:]]
    few, t.pages = t.pages, pages
    assert np.array_equal(wide(t.run(hip, bufs=tuple(far))), want)
    path = to_dev(np.array([[1, 4, 6], [0, 1, 1]], np.int32), dev)
    count = to_dev(np.array([3, 2], np.int32), dev)
    for b, n in ((near, few), (far, pages)):
        hip.kv_keep_q4_0(b[0], n, 16, b[1], t.stride, b[2], b[3], path, 3, count, 2, max(nodes), 2, 128)
    assert np.array_equal(from_dev(cache[base * page_bytes:]), from_dev(near[0].view(-1)))
    del far, cache
    torch.cuda.empty_cache()
