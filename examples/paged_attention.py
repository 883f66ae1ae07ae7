"""One attention layer that serves several requests from a paged Q4_0 cache: prompts first, then a
token each per step, with the framework's kernels from the quantizer to the residual sum.

    python examples/paged_attention.py

A step of the layer, x the f32 rows of its tokens ([token][hidden]):

    quantize_row_q8_0   x                       -> Q8_0 rows
    q8_0_q8_0_gemm      rows . fused weights    -> [token][queries | keys | values], f32
    kv_tables           lengths, free pages     -> block table, positions, slots
    rope                the queries, in place
    kv_store_q4_0       the keys (turned) and values into their slots
    attn_q4_0           the queries over the cache
    quantize_row_q8_0, q8_0_q8_0_gemm, add_f32   the output projection and the sum with x

Queries, keys and values stay columns of the fused product: the strides of a token and of a head say
where.  The lengths are known here as the scheduler knows them, so that no call waits for the device.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "tianchen-rv_amd"))
import tcrv_hip as hip  # noqa: E402

Q8_BLOCK = 34  # bytes of 32 values


def q8_rows(x):
    """f32 [rows][n] -> Q8_0 rows, n / 32 blocks each."""
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


class PagedAttention:
    def __init__(self, hidden=1024, heads=8, kv_heads=2, head_dim=128, page_size=32, pages=256,
                 requests=4, most_tokens=2048, window=0, seed=1, device="cuda:0"):
        self.hidden, self.heads, self.kv_heads, self.dim = hidden, heads, kv_heads, head_dim
        self.page_size, self.pages, self.requests, self.window = page_size, pages, requests, window
        self.device, self.most_tokens = torch.device(device), most_tokens
        gen = torch.Generator().manual_seed(seed)

        def weights(rows, n):
            w = torch.randn((rows, n), generator=gen) * n ** -0.5
            return q8_rows(w.to(self.device))

        self.w_in = weights((heads + 2 * kv_heads) * head_dim, hidden)
        self.w_out = weights(hidden, heads * head_dim)
        self.table = torch.empty((most_tokens, head_dim), device=self.device)  # pairs of cos, sin
        hip.rope_table(head_dim, self.table, most_tokens)
        page_bytes = hip.kv_q4_0_page_bytes(page_size, kv_heads, head_dim)
        self.cache = torch.empty((pages, page_bytes), dtype=torch.uint8, device=self.device)
        self.width = -(-most_tokens // page_size)
        self.block_table = torch.full((requests, self.width), -1, dtype=torch.int32,
                                      device=self.device)
        self.free = torch.arange(pages, dtype=torch.int32, device=self.device)
        self.pages_taken = 0
        # the requests' tokens so far, for the host's bounds and for the kernels
        self.lengths = np.zeros(requests, np.int64)
        self.context = torch.zeros(requests, dtype=torch.int32, device=self.device)
        self.added = (None, None)  # of the newest step, and on the device
        self.ws = torch.empty(0, dtype=torch.uint8, device=self.device)

    def step(self, x, added):
        """x: the new tokens' rows, request after request, added[r] of request r."""
        added = np.asarray(added, np.int64)
        n, ps, heads, kv, dim = len(added), self.page_size, self.heads, self.kv_heads, self.dim
        tokens, features = x.shape[0], (heads + 2 * kv) * dim
        after = self.lengths + added
        new_pages = int((-(-after // ps) - -(-self.lengths // ps)).sum())
        if self.pages_taken + new_pages > self.pages or after.max() > self.most_tokens:
            raise RuntimeError("the cache is full")

        if self.added[0] is None or not np.array_equal(self.added[0], added):
            on_device = torch.from_numpy(added.astype(np.int32)).to(self.device)
            self.added = (added, on_device)

        qkv = project(q8_rows(x), self.w_in, self.hidden).view(tokens, heads + 2 * kv, dim)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]

        def empty(count, dtype=torch.int32):
            return torch.empty(count, dtype=dtype, device=self.device)

        first, length, positions = empty(n + 1), empty(n), empty(tokens)
        slots, taken = empty(tokens, torch.int64), empty(1)
        free = self.free[self.pages_taken:]
        hip.kv_tables(self.context, self.added[1], n, ps, free, len(free), self.block_table, self.width, first, length, positions, slots, tokens, taken)
        rows = self.table.shape[0]
        hip.rope("f32", "half", q, features, dim, q, features, dim, positions, self.table, rows,
                 tokens, heads, dim, dim)
        hip.kv_store_q4_0("f32", k, features, dim, v, features, dim, "half", positions, self.table,
                          rows, dim, slots, self.cache, self.pages, ps, tokens, kv, dim)
        out = torch.empty((tokens, heads * dim), device=self.device)
        bounds = int(added.max()), int(after.max())
        need = hip.attn_q4_0_workspace_bytes("f32", n, tokens, *bounds, heads, kv, dim)
        if need > self.ws.numel():
            self.ws = empty(need, torch.uint8)
        hip.attn_q4_0("f32", q, features, dim, self.cache, self.pages, ps, self.block_table,
                      self.width, first, length, n, tokens, *bounds, heads, kv, dim, dim ** -0.5,
                      True, self.window, out, heads * dim, dim, self.ws, need)

        y = project(q8_rows(out), self.w_out, heads * dim)
        hip.add_f32(x, y, y, x.numel())
        self.lengths, self.context = after, length
        self.pages_taken += new_pages
        self.last = dict(q=q, slots=slots, attended=out)  # of the newest step
        return y


def main():
    prompts, steps = [700, 33, 1290, 256], 64
    layer = PagedAttention()
    gen = torch.Generator().manual_seed(2)
    x = torch.randn((sum(prompts), layer.hidden), generator=gen).to(layer.device)
    y = layer.step(x, prompts)
    last = [sum(prompts[:r + 1]) - 1 for r in range(len(prompts))]
    x = y[last]
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(-8, steps):  # the first ones untimed
        if i == 0:
            begin.record()
        x = layer.step(x.contiguous(), [1] * len(prompts))
        x = x / x.norm(dim=-1, keepdim=True) * layer.hidden ** 0.5
    end.record()
    torch.cuda.synchronize()
    print(f"{len(prompts)} requests, prompts of {prompts} tokens, {steps} steps: "
          f"{begin.elapsed_time(end) / steps * 1e3:.0f} us a step, {layer.pages_taken} pages of "
          f"{layer.page_size} tokens in use, lengths {layer.lengths.tolist()}")


if __name__ == "__main__":
    main()
