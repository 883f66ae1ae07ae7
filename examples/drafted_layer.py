"""One layer of a model that checks drafted tokens: several requests over a paged Q4_0 cache, their prompts
first, then a tree of drafted tokens each per step, of which a path is kept, with the framework's kernels
from norm to norm.

    python examples/drafted_layer.py

A step of the layer, x the f32 rows of its tokens ([token][hidden]):

    add_rms_norm        x                       -> Q8_0 rows
    q8_0_q8_0_gemm      rows . fused weights    -> [token][queries | keys | values], f32
    kv_tables           lengths, free pages     -> block table, positions, slots
    tree_tables         parents                 -> ancestors, positions by depth
    rope                the queries, in place
    kv_store_q4_0       the keys (turned) and values into their slots
    attn_tree_q4_0      the queries over the cache, each node over its ancestors
    quantize_row_q8_0, q8_0_q8_0_gemm           the output projection
    add_rms_norm        its sum with x, and that sum's norm -> Q8_0 rows
    gated_q4_0_q8_0     rows . gate, up (Q4_0)  -> Q8_0 rows
    q8_0_q8_0_gemm, add_f32                     the down projection and the sum

After a model's last layer the accepted path is known, and in every layer

    kv_keep_q4_0        the path's keys and values to follow the cached tokens

Prompts go the same way with attn_q4_0.  Trees, paths and lengths are known here as the scheduler knows
them, so that nothing is read back from the device.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "tianchen-rv_amd"))
import tcrv_hip as hip  # noqa: E402

Q4_BLOCK, Q8_BLOCK = 18, 34  # bytes of 32 values
EPS = 1e-5


def q4_rows(x):
    """f32 [rows][n] -> Q4_0 rows: a scale and sixteen bytes of two quants for 32 values."""
    blocks = x.view(x.shape[0], -1, 32)
    d = (blocks.abs().amax(-1, keepdim=True) / 7).half()
    quants = (blocks / d.float().clamp(min=1e-7)).round().clamp(-8, 7).add(8).to(torch.uint8)
    packed = torch.cat((d.view(torch.uint8), quants[..., :16] | quants[..., 16:] << 4), -1)
    return packed.view(x.shape[0], -1)


def q8_rows(x):
    """f32 [rows][n] -> Q8_0 rows."""
    rows, n = x.shape
    out = torch.empty((rows, n // 32 * Q8_BLOCK), dtype=torch.uint8, device=x.device)
    hip.quantize_row_q8_0(rows * n, x, out)
    return out


def project(rows, weights, n):
    """[token][feature] = rows . weights, both Q8_0 rows of n values."""
    tokens, features = rows.shape[0], weights.shape[0]
    out = torch.empty((tokens, features), device=rows.device)
    hip.q8_0_q8_0_gemm(n, out, rows, weights, weights.shape[1], tokens, features, rows.shape[1],
                       features)
    return out


class DraftedLayer:
    def __init__(self, hidden=1024, wide=2816, heads=8, kv_heads=2, head_dim=128, page_size=32,
                 pages=256, requests=4, most_tokens=2048, window=0, seed=1, device="cuda:0"):
        self.hidden, self.wide, self.heads, self.kv_heads, self.dim = hidden, wide, heads, kv_heads, head_dim
        self.page_size, self.pages, self.requests, self.window = page_size, pages, requests, window
        self.device, self.most_tokens = torch.device(device), most_tokens
        gen = torch.Generator().manual_seed(seed)

        def random(rows, n):
            return (torch.randn((rows, n), generator=gen) * n ** -0.5).to(self.device)

        self.w_in = q8_rows(random((heads + 2 * kv_heads) * head_dim, hidden))
        self.w_out = q8_rows(random(hidden, heads * head_dim))
        self.gate, self.up = q4_rows(random(wide, hidden)), q4_rows(random(wide, hidden))
        self.w_down = q8_rows(random(hidden, wide))
        self.norm_in, self.norm_out = (1 + random(1, hidden)[0] for _ in range(2))
        self.table = torch.empty((most_tokens, head_dim), device=self.device)  # pairs of cos, sin
        hip.rope_table(head_dim, self.table, most_tokens)
        page_bytes = hip.kv_q4_0_page_bytes(page_size, kv_heads, head_dim)
        self.cache = torch.empty((pages, page_bytes), dtype=torch.uint8, device=self.device)
        self.width = -(-most_tokens // page_size)
        self.block_table = torch.full((requests, self.width), -1, dtype=torch.int32,
                                      device=self.device)
        self.free = torch.arange(pages, dtype=torch.int32, device=self.device)
        # the requests' cached tokens, for the host's bounds and for the kernels
        self.lengths = np.zeros(requests, np.int64)
        self.context = torch.zeros(requests, dtype=torch.int32, device=self.device)
        self.ws = torch.empty(0, dtype=torch.uint8, device=self.device)

    def _ints(self, values):
        return torch.from_numpy(np.ascontiguousarray(values, np.int32)).to(self.device)

    def _empty(self, *shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device=self.device)

    def step(self, x, added, parents=None):
        """x: the new tokens' rows, request after request, added[r] of request r: a prompt's next ones, or
        a tree's nodes, parents[r][i] the parent of node i (below i; -1: it follows the cached tokens).
        The tokens are cached; keep() says which nodes stay."""
        added = np.asarray(added, np.int64)
        n, ps, heads, kv, dim = len(added), self.page_size, self.heads, self.kv_heads, self.dim
        tokens, features, wide = x.shape[0], (heads + 2 * kv) * dim, self.wide
        before, after = self.lengths, self.lengths + added
        new_pages = int((-(-after // ps) - -(-before // ps)).sum())
        if new_pages > len(self.free) or after.max() > self.most_tokens:
            raise RuntimeError("the cache is full")

        rows = self._empty(tokens, self.hidden // 32 * Q8_BLOCK, dtype=torch.uint8)
        hip.add_rms_norm("f32", x, self.hidden, None, 0, None, 0, self.norm_in, EPS, None, 0, rows,
                         rows.shape[1], tokens, self.hidden)
        qkv = project(rows, self.w_in, self.hidden).view(tokens, heads + 2 * kv, dim)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]

        first, length, positions = self._empty(n + 1), self._empty(n), self._empty(tokens)
        slots, taken = self._empty(tokens, dtype=torch.int64), self._empty(1)
        hip.kv_tables(self.context, self._ints(added), n, ps, self.free, len(self.free),
                      self.block_table, self.width, first, length, positions, slots, tokens, taken)
        if parents is not None:
            words = max(1, -(-int(added.max()) // 64))
            ancestors = self._empty(tokens, words, dtype=torch.int64)
            hip.tree_tables(self._ints(np.concatenate([np.asarray(p, np.int32) for p in parents])),
                            first, length, n, ancestors, words, positions, tokens)
        turns = self.table.shape[0]
        hip.rope("f32", "half", q, features, dim, q, features, dim, positions, self.table, turns,
                 tokens, heads, dim, dim)
        hip.kv_store_q4_0("f32", k, features, dim, v, features, dim, "half", positions, self.table,
                          turns, dim, slots, self.cache, self.pages, ps, tokens, kv, dim)
        attended = self._empty(tokens, heads * dim, dtype=torch.float32)
        bounds = int(added.max()), int(after.max())
        size = hip.attn_q4_0_workspace_bytes if parents is None else hip.attn_tree_q4_0_workspace_bytes
        need = size("f32", n, tokens, *bounds, heads, kv, dim)
        if need > self.ws.numel():
            self.ws = self._empty(need, dtype=torch.uint8)
        cached = (q, features, dim, self.cache, self.pages, ps, self.block_table, self.width, first, length)
        to = (self.window, attended, heads * dim, dim, self.ws, need)
        if parents is None:
            hip.attn_q4_0("f32", *cached, n, tokens, *bounds, heads, kv, dim, dim ** -0.5, True, *to)
        else:
            hip.attn_tree_q4_0("f32", *cached, ancestors, words, n, tokens, *bounds, heads, kv, dim,
                               dim ** -0.5, *to)

        y = project(q8_rows(attended), self.w_out, heads * dim)
        total = torch.empty_like(x)
        hip.add_rms_norm("f32", y, self.hidden, x, self.hidden, total, self.hidden, self.norm_out, EPS,
                         None, 0, rows, rows.shape[1], tokens, self.hidden)
        inner = self._empty(tokens, wide // 32 * Q8_BLOCK, dtype=torch.uint8)
        hip.gated_q4_0_q8_0("f32", "silu", self.hidden, None, 0, inner, inner.shape[1], self.gate,
                            self.up, self.gate.shape[1], rows, rows.shape[1], wide, tokens)
        y = project(inner, self.w_down, wide)
        hip.add_f32(total, y, y, y.numel())

        self.free = self.free[new_pages:]
        self.lengths, self.before = after, (before, self.context)
        self.context = length
        self.last = dict(first=first, length=length, added=added, q=q, attended=attended, total=total,
                         rows=rows, inner=inner)  # of the newest step
        return y

    def keep(self, paths):
        """Of the newest step's nodes those of paths[r] stay, from the tree's top downwards."""
        before, context = self.before
        kv, ps, last = self.kv_heads, self.page_size, self.last
        count = np.array([len(p) for p in paths], np.int64)
        path = np.zeros((len(paths), max(1, int(count.max()))), np.int32)
        for r, p in enumerate(paths):
            path[r, :len(p)] = p
        counts = self._ints(count)
        hip.kv_keep_q4_0(self.cache, self.pages, ps, self.block_table, self.width, last["first"],
                         last["length"], self._ints(path), path.shape[1], counts, len(paths),
                         int(last["added"].max()), kv, self.dim)
        self.context = torch.empty_like(context)
        hip.add_i32(context, counts, self.context, len(paths))
        kept = before + count
        spare = [self.block_table[r, -(-kept[r] // ps):-(-self.lengths[r] // ps)]
                 for r in range(len(paths))]
        self.free = torch.cat([*spare, self.free])
        self.lengths = kept


def random_tree(rng, nodes):
    """Parents of a tree, each node's a random earlier one of the newest four."""
    return [rng.integers(max(-1, i - 4), i) for i in range(nodes)]


def random_path(rng, tree):
    """The nodes from the top to a random one."""
    path, at = [], rng.integers(len(tree))
    while at >= 0:
        path.insert(0, int(at))
        at = tree[at]
    return path


def main():
    prompts, nodes, steps = [700, 33, 1290, 256], 12, 64
    layer = DraftedLayer()
    rng, gen = np.random.default_rng(2), torch.Generator().manual_seed(2)
    layer.step(torch.randn((sum(prompts), layer.hidden), generator=gen).to(layer.device), prompts)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    drafted = torch.randn((len(prompts) * nodes, layer.hidden), generator=gen).to(layer.device)
    kept = 0
    for i in range(-8, steps):  # the first ones untimed
        if i == 0:
            begin.record()
            kept = int(layer.lengths.sum())
        trees = [random_tree(rng, nodes) for _ in prompts]
        layer.step(drafted, [nodes] * len(prompts), trees)
        layer.keep([random_path(rng, tree) for tree in trees])
    end.record()
    torch.cuda.synchronize()
    print(f"{len(prompts)} requests, prompts of {prompts} tokens, {steps} steps of {nodes} drafted tokens "
          f"each: {begin.elapsed_time(end) / steps * 1e3:.0f} us a step, "
          f"{(int(layer.lengths.sum()) - kept) / steps / len(prompts):.1f} tokens kept a step and request, "
          f"{layer.pages - len(layer.free)} pages of {layer.page_size} tokens in use, lengths "
          f"{layer.lengths.tolist()}")


if __name__ == "__main__":
    main()
