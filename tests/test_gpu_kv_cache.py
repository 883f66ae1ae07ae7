"""The paged Q4_0 cache's operators on the GPU against their plain forms (tests/kv_plain.py): tables
and stored bytes exactly, rotations bit for bit in f32, attention against float64."""
import numpy as np
import pytest
import torch

import kv_plain
import synth
from gpu_util import from_dev, to_dev

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev_rows(x, elem, dev):
    """float32 values (already rounded to elem) as a device tensor of that type."""
    return to_dev(x, dev).to(TORCH[elem])


def wide(t):
    return from_dev(t.float())


# ---------------------------------------------------------------- tables ---

@pytest.mark.parametrize("requests,page,context,added,spare,stride_cut,token_cut", [
    (1, 16, 0, 1, 5, 0, 0),
    (1, 16, 16, 1, 5, 0, 0),
    (3, 16, 100, 40, 3, 0, 0),
    (64, 64, 4096, 1, 9, 0, 0),
    (256, 16, 50, 30, 1, 0, 0),
    (257, 48, 200, 90, 0, 0, 7),        # two runs of requests; more tokens than max_tokens
    (700, 32, 300, 3, 2, 0, -50),       # room for more tokens than there are
    (40, 16, 200, 100, -25, 0, 0),      # free pages run out
    (30, 16, 200, 100, 4, 3, 0),        # table rows too short
    (5, 17, 60, 33, 4, 0, 0),           # a page size that the cache does not have
    (1, 1, 0, 5000, 0, 0, 0),
])
def test_tables(hip, dev, requests, page, context, added, spare, stride_cut, token_cut):
    rng = np.random.default_rng(requests * 1000 + page)
    c = rng.integers(0, context + 1, requests).astype(np.int32)
    a = rng.integers(0, added + 1, requests).astype(np.int32)
    c[0], a[0] = context, added
    if requests > 4:
        a[2] = -3
        c[3] = -7
    cc, aa = np.maximum(c, 0), np.maximum(a, 0)
    held, need = -(-cc // page), -(-(cc + aa) // page)
    stride = max(1, int(need.max()) + 1 - stride_cut)
    ids = rng.permutation(int(need.sum()) + 50).astype(np.int32)
    free = ids[:max(0, int((need - held).sum()) + spare)]
    table = np.full((requests, stride), -9, np.int32)
    for r in range(requests):
        n = min(int(held[r]), stride)
        table[r, :n] = rng.integers(0, 10000, n)
        if n and r % 7 == 3:
            table[r, n - 1] = -1  # a page that was missing a step before
    max_tokens = max(0, int(aa.sum()) - token_cut)
    want = kv_plain.tables(c, a, page, free, table, max_tokens)
    got_table = to_dev(table, dev)
    made = {k: torch.full((n,), -77, dtype=t, device=dev) for k, n, t in (
        ("first", requests + 1, torch.int32), ("length", requests, torch.int32),
        ("positions", max(max_tokens, 1), torch.int32), ("slots", max(max_tokens, 1), torch.int64),
        ("taken", 1, torch.int32))}
    dc, da, df = to_dev(c, dev), to_dev(a, dev), to_dev(np.append(free, np.int32(0)).astype(np.int32), dev)
    for _ in range(2):  # the second time over its own results
        hip.kv_tables(dc, da, requests, page, df, len(free), got_table, stride, made["first"],
                      made["length"], made["positions"], made["slots"], max_tokens, made["taken"])
        assert np.array_equal(from_dev(got_table), want["block_table"])
        for k in made:
            got = from_dev(made[k])
            assert np.array_equal(got[:max_tokens] if k in ("positions", "slots") else got,
                                  want[k]), k


def test_tables_of_nothing(hip, dev):
    first, taken = (torch.full((1,), 5, dtype=torch.int32, device=dev) for _ in range(2))
    slots = torch.full((3,), 5, dtype=torch.int64, device=dev)
    positions = torch.full((3,), 5, dtype=torch.int32, device=dev)
    hip.kv_tables(None, None, 0, 16, None, 0, None, 0, first, None, positions, slots, 3, taken)
    assert from_dev(first)[0] == 0 and from_dev(taken)[0] == 0
    assert (from_dev(slots) == -1).all() and (from_dev(positions) == -1).all()


def test_tables_saturate(hip, dev):
    big = 2 ** 31 - 1
    c, a = to_dev(np.array([big, 1], np.int32), dev), to_dev(np.array([big, big], np.int32), dev)
    table = torch.full((2, 2), -5, dtype=torch.int32, device=dev)
    first = torch.zeros(3, dtype=torch.int32, device=dev)
    length = torch.zeros(2, dtype=torch.int32, device=dev)
    taken = torch.zeros(1, dtype=torch.int32, device=dev)
    positions = torch.zeros(4, dtype=torch.int32, device=dev)
    slots = torch.zeros(4, dtype=torch.int64, device=dev)
    hip.kv_tables(c, a, 2, 16, to_dev(np.array([4], np.int32), dev), 1, table, 2, first, length,
                  positions, slots, 4, taken)
    assert from_dev(first).tolist() == [0, big, big] and from_dev(length).tolist() == [big, big]
    assert from_dev(table).tolist() == [[-5, -5], [-5, 4]] and from_dev(taken)[0] == 1
    assert (from_dev(slots) == -1).all()


# ------------------------------------------------------------------ rope ---

@pytest.mark.parametrize("scaling,n,kw", [
    ("none", 128, {}), ("none", 2, {}), ("linear", 64, dict(factor=4.0)),
    ("ntk", 96, dict(factor=8.0)), ("yarn", 128, dict(factor=16.0)),
    ("yarn", 64, dict(factor=4.0, trained_context=8192.0, beta_fast=16.0, beta_slow=2.0,
                      base=500000.0)),
    ("none", 128, dict(divisors=True)), ("none", 64, dict(amplitude=1.25)),
])
def test_rope_table(hip, dev, scaling, n, kw):
    """Angles reach 2^18 here; f64 angles differ by some 2^-52 of that, the f32 result is rounded
    once (2^-25 of at most 1.3): 1e-7 is above both."""
    kw = dict(kw)
    divisors = np.linspace(1.0, 8.0, n // 2).astype(np.float32) if kw.pop("divisors", 0) else None
    first, count = 262100, 37
    plain = {k: v for k, v in kw.items() if k not in ("amplitude", "trained_context")}
    angles, amplitude = kv_plain.rope_angles(
        n, np.arange(first, first + count), plain.pop("base", 10000.0), scaling,
        trained=kw.get("trained_context", 4096.0), divisors=divisors, **plain)
    amplitude = kw.get("amplitude", amplitude)
    table = torch.full((count + 1, n // 2, 2), 7.0, device=dev)
    hip.rope_table(n, table, count, first, scaling=scaling,
                   divisors=None if divisors is None else to_dev(divisors, dev), **kw)
    got = from_dev(table)
    assert (got[count] == 7.0).all()
    want = np.stack([np.cos(angles), np.sin(angles)], -1) * amplitude
    assert np.abs(got[:count] - want).max() <= 1e-7


def plain_table(n, rows):
    a, _ = kv_plain.rope_angles(n, np.arange(rows), 10000.0)
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


@pytest.mark.parametrize("elem", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,n,pad,off", [
    (5, 3, 128, 128, 0, 0), (7, 32, 128, 64, 0, 0), (3, 2, 80, 20, 0, 0), (2, 5, 64, 2, 0, 0),
    (4, 3, 64, 64, 4, 1), (3, 2, 33, 10, 1, 0), (2, 1, 256, 256, 0, 0), (1, 64, 192, 96, 8, 0),
    (3, 2, 16, 0, 0, 0), (1100, 3, 64, 64, 0, 0), (2, 2, 4096, 4096, 0, 0),
])
def test_rope(hip, dev, elem, layout, tokens, heads, dim, n, pad, off):
    """Bit for bit in f32 steps; strides beyond the rows, addresses off the 16-byte grid, positions
    outside the table, in place and apart, forward and inverse."""
    rng = np.random.default_rng(tokens * dim + n)
    x = kv_plain.round_to(rng.standard_normal((tokens, heads, dim)), elem)
    table = plain_table(max(n, 2), 50)[:, :n // 2] if n else np.zeros((50, 0, 2), np.float32)
    positions = rng.integers(0, 50, tokens).astype(np.int32)
    if tokens > 2:
        positions[1], positions[2] = -1, 50
    xs, ys = dim + pad, dim + 2 * pad
    src = torch.full((tokens * heads * xs + off,), 3.0, dtype=TORCH[elem], device=dev)
    src[off:].view(tokens, heads, xs)[..., :dim] = dev_rows(x, elem, dev)
    dt, dp = to_dev(table, dev) if n else None, to_dev(positions, dev)
    for inverse in (False, True):
        want = kv_plain.round_to(kv_plain.rope(x, positions, table, n, layout, inverse), elem)
        out = torch.full((tokens * heads * ys + off,), 5.0, dtype=TORCH[elem], device=dev)
        hip.rope(elem, layout, src[off:], heads * xs, xs, out[off:], heads * ys, ys, dp, dt, 50,
                 tokens, heads, dim, n, inverse)
        got = wide(out)[off:].reshape(tokens, heads, ys)
        assert np.array_equal(got[..., :dim].view(np.uint32), want.view(np.uint32))
        assert (got[..., dim:] == 5.0).all() and (wide(out)[:off] == 5.0).all()
        same = src.clone()
        hip.rope(elem, layout, same[off:], heads * xs, xs, same[off:], heads * xs, xs, dp, dt, 50,
                 tokens, heads, dim, n, inverse)
        got = wide(same)[off:].reshape(tokens, heads, xs)
        assert np.array_equal(got[..., :dim].view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_inverse_is_the_gradient(hip, dev, layout):
    """sum(g . turn(x)) by differences in x against the inverse turn of g.  The turn is linear, so a
    difference of any step is exact but for f32 rounding: values of at most 6, products of three
    roundings, 2^-24 each, over a step of 1: 6e-6 is above it."""
    rng = np.random.default_rng(3)
    x, g = (rng.standard_normal((4, 2, 64)).astype(np.float32) for _ in range(2))
    table, positions = plain_table(48, 90), np.array([0, 3, 88, 41], np.int32)
    dt, dp = to_dev(table, dev), to_dev(positions, dev)

    def turn(v, inverse=False):
        out = torch.empty(4, 2, 64, device=dev)
        hip.rope("f32", layout, to_dev(v, dev), 128, 64, out, 128, 64, dp, dt, 90, 4, 2, 64, 48,
                 inverse)
        return from_dev(out).astype(np.float64)

    grad, base = turn(g, True), turn(x)
    for e in (0, 1, 23, 24, 31, 47, 48, 63):
        up = x.copy()
        up[..., e] += 1.0
        step = (up[..., e] - x[..., e]).astype(np.float64)
        diff = (g * (turn(up) - base)).sum(-1) / step
        assert np.abs(diff - grad[..., e]).max() <= 6e-6 * 64 ** 0.5


# ------------------------------------------------------- store and load ---

@pytest.mark.parametrize("elem", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout,tokens,heads,dim,page,n,apart", [
    ("half", 1, 1, 64, 16, 64, 0), ("interleaved", 37, 2, 128, 16, 128, 0),
    ("half", 70, 3, 128, 48, 128, 0), ("half", 21, 2, 192, 32, 96, 1),
    ("interleaved", 9, 1, 256, 64, 30, 1), ("half", 9, 2, 64, 16, 6, 0),
    ("half", 33, 2, 256, 16, 0, 0),
])
def test_store_and_load(hip, dev, elem, layout, tokens, heads, dim, page, n, apart):
    """The cache's bytes as ggml's quantizer makes them of the turned keys, at the layout's places,
    and nothing else written; read back as the values they stand for.  `apart`: rows a little apart,
    off the 16-byte grid."""
    rng = np.random.default_rng(tokens * dim + page)
    k, v = (kv_plain.round_to(rng.standard_normal((tokens, heads, dim)) * 3, elem)
            for _ in range(2))
    k[0, 0, :32] = 0.0                       # an empty block
    k[0, 0, 32:64] = kv_plain.round_to(np.full(32, -1.5), elem)  # ties: the first counts
    v[0, 0, 32:64] = kv_plain.round_to(np.where(np.arange(32) % 2, 2.0, -2.0), elem)
    v[tokens - 1, 0, :32] *= kv_plain.round_to(np.float32(2.0 ** -13), elem)  # subnormal scales
    v = kv_plain.round_to(v, elem)
    pages = -(-tokens // page) + 2
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 8:
        slots[3], slots[5], slots[7] = -1, pages * page, 1 << 40
    table = plain_table(n, 60) if n else np.zeros((1, 0, 2), np.float32)
    positions = rng.integers(0, 60, tokens).astype(np.int32)
    if tokens > 8:
        positions[2] = 60
    turned = kv_plain.rope(k, positions, table, n, layout)
    want = kv_plain.Cache(pages, page, heads, dim)
    want.store(slots, kv_plain.quantize(turned), kv_plain.quantize(v))
    assert hip.kv_q4_0_page_bytes(page, heads, dim) == want.bytes[0].size
    cache = torch.full((want.bytes.size,), 0xFF, dtype=torch.uint8, device=dev)
    if apart:
        rows = torch.zeros(tokens, 2 * heads, dim + 1, dtype=TORCH[elem], device=dev)
        rows[:, :heads, :dim], rows[:, heads:, :dim] = (dev_rows(x, elem, dev) for x in (k, v))
        dk, dv = rows[:, :heads], rows[:, heads:]
    else:
        dk, dv = dev_rows(k, elem, dev), dev_rows(v, elem, dev)
    ds = to_dev(slots, dev)
    hip.kv_store_q4_0(elem, dk, dk.stride(0), dk.stride(1), dv, dv.stride(0), dv.stride(1), layout,
                      to_dev(positions, dev) if n else None, to_dev(table, dev) if n else None,
                      60, n, ds, cache, pages, page, tokens, heads, dim)
    got = from_dev(cache).reshape(want.bytes.shape)
    assert np.array_equal(got, want.bytes)

    for to in ("f32", elem):
        step = dim + apart
        out = torch.full((2, tokens, heads, step), 9.0, dtype=TORCH[to], device=dev)
        hip.kv_load_q4_0(to, cache, pages, page, ds, out[0], heads * step, step, out[1],
                         heads * step, step, tokens, heads, dim)
        back = wide(out)
        assert (back[..., dim:] == 9.0).all()
        for which, x in ((0, turned), (1, v)):
            ref = kv_plain.values(*kv_plain.quantize(x)).astype(np.float32)
            ref[(slots < 0) | (slots >= pages * page)] = 0.0
            assert np.array_equal(back[which][..., :dim], kv_plain.round_to(ref, to))


def test_store_of_what_is_not_finite(hip, dev):
    """A NaN makes its block's scale NaN and no other; an infinity, or more than fp16 holds, makes
    it infinite."""
    k = np.ones((1, 1, 128), np.float32)
    k[0, 0, 5], k[0, 0, 40], k[0, 0, 70] = np.nan, np.inf, 1e6
    v = np.ones((1, 1, 128), np.float32)
    cache = torch.zeros(16 * 144, dtype=torch.uint8, device=dev)
    slot = torch.zeros(1, dtype=torch.int64, device=dev)
    hip.kv_store_q4_0("f32", to_dev(k, dev), 128, 128, to_dev(v, dev), 128, 128, "half", None,
                      None, 0, 0, slot, cache, 1, 16, 1, 1, 128)
    got = from_dev(cache)
    d = got[16 * 64:16 * 64 + 32].view(np.float16).reshape(4, 4)[:, 0]
    assert np.isnan(d[0]) and np.isinf(d[1]) and np.isinf(d[2]) and d[3] == -0.125
    out = torch.empty(2, 1, 1, 128, device=dev)
    hip.kv_load_q4_0("f32", cache, 1, 16, slot, out[0], 128, 128, out[1], 128, 128, 1, 1, 128)
    assert (from_dev(out)[1] == 1.0).all() and (from_dev(out)[0, 0, 0, 96:] == 1.0).all()


# ------------------------------------------------------------- attention ---

class Setup:
    """Requests with random rows, their tokens in shuffled pages; all else in the cache is 0xff:
    NaN scales."""

    def __init__(self, dev, elem, lengths, added, heads, kv, dim, page, seed=0, spread=1.0,
                 values=1.0, stride=None):
        rng = np.random.default_rng(seed + 17 * dim + page)
        self.dev, self.elem, self.heads, self.kv, self.dim, self.page = (dev, elem, heads, kv, dim,
                                                                         page)
        self.lengths, self.added = np.array(lengths, np.int32), np.array(added, np.int32)
        n = len(lengths)
        self.stride = stride or max(1, max(-(-x // page) for x in lengths))
        total = sum(-(-x // page) for x in lengths)
        self.pages = total + 3
        ids = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((n, self.stride), 2 ** 30, np.int32)
        cache = kv_plain.Cache(self.pages, page, kv, dim)
        self.k, self.v, at = [], [], 0
        for r, length in enumerate(lengths):
            blocks = -(-length // page)
            self.table[r, :blocks] = ids[at:at + blocks]
            at += blocks
            kq = kv_plain.quantize(rng.standard_normal((length, kv, dim)).astype(np.float32))
            vq = kv_plain.quantize((values * rng.standard_normal((length, kv, dim)))
                                   .astype(np.float32))
            t = np.arange(length)
            slots = self.table[r, t // page].astype(np.int64) * page + t % page
            self.slots = slots
            self._put(cache, slots, kq, vq)
            self.k.append(kv_plain.values(*kq))
            self.v.append(kv_plain.values(*vq))
        self.cache = cache
        self.first = np.concatenate([[0], np.cumsum(self.added)]).astype(np.int32)
        self.tokens = int(self.first[-1])
        self.q = kv_plain.round_to(spread * rng.standard_normal((self.tokens, heads, dim)), elem)

    @staticmethod
    def _put(cache, slots, kq, vq):
        """Cache.store by whole arrays (test_store_and_load pins the two to one layout)."""
        heads, nb, ps = cache.heads, cache.nb, cache.page_size
        page, t = slots // ps, slots % ps
        h = np.arange(heads)[None, :]
        at, big = (page[:, None], h), cache.bytes
        tt = t[:, None]
        for b in range(nb):
            for j in range(16):
                big[at + ((tt * 4 + j // 4) * nb * 4 + b * 4 + j % 4,)] = kq[1][:, :, b, j]
                o = (((tt // 4) * 16 + j) * (nb // 2) + b // 2) * 8 + (tt % 4) * 2 + b % 2
                big[at + (cache.quants + cache.scales + o,)] = vq[1][:, :, b, j]
            o = ((tt // 4) * nb + b) * 8 + (tt % 4) * 2
            for which, base in ((kq, cache.quants), (vq, 2 * cache.quants + cache.scales)):
                pair = np.ascontiguousarray(which[0][:, :, b]).view(np.uint8).reshape(len(t), heads,
                                                                                     2)
                for i in range(2):
                    big[at + (base + o + i,)] = pair[:, :, i]

    def run(self, hip, scale=None, causal=True, window=0, q=None, out=None, max_added=None,
            max_length=None, tokens=None, stream=None, table=None, bufs=None):
        elem, heads, kv, dim = self.elem, self.heads, self.kv, self.dim
        scale = dim ** -0.5 if scale is None else scale
        n, tokens = len(self.lengths), tokens or self.tokens
        q = dev_rows(self.q, elem, self.dev) if q is None else q
        out = torch.full((tokens, heads, dim), 3.0, dtype=TORCH[elem], device=self.dev) \
            if out is None else out
        most_a = int(self.added.max()) if max_added is None else max_added
        most_l = int(self.lengths.max()) if max_length is None else max_length
        need = hip.attn_q4_0_workspace_bytes(elem, n, tokens, most_a, most_l, heads, kv, dim)
        ws = torch.full((max(need // 4, 4),), float("nan"), device=self.dev)
        table = self.table if table is None else table
        b = bufs or self.buffers(table)
        hip.attn_q4_0(elem, q, q.stride(0), q.stride(1), b[0], self.pages, self.page, b[1],
                      self.stride, b[2], b[3], n, tokens, most_a, most_l, heads, kv, dim, scale,
                      causal, window, out, out.stride(0), out.stride(1), ws, need, stream)
        return out

    def buffers(self, table=None):
        table = self.table if table is None else table
        return (to_dev(self.cache.bytes.reshape(-1), self.dev), to_dev(table, self.dev),
                to_dev(self.first, self.dev), to_dev(self.lengths, self.dev))

    def want(self, scale=None, causal=True, window=0):
        scale = np.float64(np.float32(self.dim ** -0.5 if scale is None else scale))
        got = [kv_plain.attend(self.q[self.first[r]:self.first[r + 1]], self.k[r], self.v[r],
                               int(self.lengths[r]) - int(self.added[r]), scale, causal, window)
               for r in range(len(self.lengths))]
        return np.concatenate(got) if got else np.zeros((0, self.heads, self.dim))

    def tolerance(self, want, scale=None):
        """A score is off by at most 2^-22 |q||k| (the queries' parts and the sums' roundings, 2^-24
        each over a dozen steps) and a weight by that and the exponential's 2^-22; the output by
        twice that of the largest value, and by its own rounding.  f16 weights add 2^-11 of it."""
        scale = self.dim ** -0.5 if scale is None else abs(scale)
        top = max([np.abs(v).max() for v in self.v if v.size] + [0.0])
        qn = np.linalg.norm(self.q.astype(np.float64), axis=-1).max() if self.q.size else 0.0
        kn = max([np.linalg.norm(k, axis=-1).max() for k in self.k if k.size] + [0.0])
        tol = 2 * top * (2.0 ** -21 * scale * qn * kn + 2.0 ** -20)
        if self.elem != "f32":
            tol += top * 2.0 ** -10 + np.abs(want) * (2.0 ** -11 if self.elem == "f16"
                                                      else 2.0 ** -8)
        return tol

    def check(self, hip, **kw):
        out = wide(self.run(hip, **kw))
        kw = {k: v for k, v in kw.items() if k in ("scale", "causal", "window")}
        want = self.want(**kw)
        scale = kw.get("scale")
        off = np.abs(out - want)
        assert np.isfinite(out).all()
        assert (off <= self.tolerance(want, scale)).all(), off.max()
        return out


ELEMS = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("lengths,added,heads,kv,dim,page", [
    ([1], [1], 1, 1, 64, 16),
    ([1, 2, 15, 16, 17], [1] * 5, 4, 1, 64, 16),
    ([31, 32, 33, 63, 64, 65, 127, 128, 129], [1] * 9, 8, 2, 128, 16),
    ([5, 530, 97], [1, 1, 1], 32, 8, 128, 48),
    ([300, 1000], [1, 1], 14, 2, 64, 32),
    ([77, 200], [1, 1], 4, 4, 192, 16),
    ([200, 40], [1, 1], 8, 1, 256, 64),
    ([100], [1], 40, 1, 128, 16),             # more queries of one kv head than a tile has rows
    ([2100, 40], [1, 1], 8, 2, 64, 16),       # split over work-groups and joined
    ([9000], [1], 4, 1, 128, 128),
    ([50, 0, 60], [3, 0, 1], 6, 2, 128, 16),  # a request without tokens
    ([0, 9], [1, 1], 2, 1, 64, 16),           # a new token that is not in the cache: sees none
    ([40, 90], [7, 2], 8, 2, 128, 16),        # several new tokens
    ([20, 33], [20, 33], 3, 1, 64, 16),       # prompts
    ([150], [150], 2, 2, 128, 32),
    ([260, 70], [130, 70], 6, 1, 64, 48),
])
def test_attention(hip, dev, elem, lengths, added, heads, kv, dim, page):
    s = Setup(dev, elem, lengths, added, heads, kv, dim, page)
    s.check(hip)
    s.check(hip, causal=False)
    s.check(hip, window=19)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("window", [1, 16, 100, 2 ** 40])
@pytest.mark.parametrize("causal", [True, False])
def test_windows(hip, dev, elem, window, causal):
    s = Setup(dev, elem, [700, 90, 3000], [1, 40, 5], 4, 2, 64, 16, seed=4)
    s.check(hip, window=window, causal=causal)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("share", [1, 2, 5, 16, 17])
def test_head_layouts(hip, dev, elem, dim, share):
    s = Setup(dev, elem, [45, 161], [2, 33], 2 * share, 2, dim, 16, seed=share)
    s.check(hip)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("values", [1e-6, 1e-3, 40.0, 3e4])
def test_value_magnitudes(hip, dev, elem, values):
    """Scales from fp16's subnormals up to its largest, below and over the bound where the weights'
    shift changes."""
    s = Setup(dev, elem, [300, 150], [1, 40], 4, 2, 128, 16, values=values)
    out = wide(s.run(hip))
    want = s.want()
    # an f16 output's own spacing where it is subnormal
    tol = s.tolerance(want) + (2.0 ** -25 if elem == "f16" else 0.0)
    held = np.abs(want) < (6e4 if elem == "f16" else np.inf)  # what the type holds
    with np.errstate(invalid="ignore"):
        assert (np.abs(out - want) <= tol)[held].all()


def test_value_scales_of_both_kinds(hip, dev):
    """Small values first and large ones late in the context, and the other way round."""
    for order in (1, -1):
        s = Setup(dev, "f32", [900], [1], 4, 1, 64, 16, values=1.0)
        big = kv_plain.quantize((300.0 * np.random.default_rng(1).standard_normal((900, 1, 64)))
                                .astype(np.float32))
        t = np.arange(900)
        late = (t >= 600) if order > 0 else (t < 200)
        kq = kv_plain.quantize(s.k[0].astype(np.float32))
        keep = kv_plain.values(*kq)
        s._put(s.cache, s.slots[late], [x[late] for x in kq], [x[late] for x in big])
        s._put(s.cache, s.slots[~late], [x[~late] for x in kq],
               [x[~late] for x in kv_plain.quantize(s.v[0].astype(np.float32))])
        s.k = [keep]
        s.v = [np.where(late[:, None, None], kv_plain.values(*big),
                        kv_plain.values(*kv_plain.quantize(s.v[0].astype(np.float32))))]
        s.check(hip)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-8, 3.0])
def test_scales(hip, dev, elem, scale):
    """None of the scores, turned round, all alike, and spread far apart."""
    s = Setup(dev, elem, [400, 33], [1, 20], 4, 2, 64, 16)
    s.check(hip, scale=scale)


def test_query_magnitudes(hip, dev):
    """The queries' power of two: rows of very small and very large values, with the scale that
    brings their scores back."""
    for spread in (2.0 ** -60, 2.0 ** 60):
        s = Setup(dev, "f32", [200], [3], 4, 2, 64, 16, spread=spread)
        s.check(hip, scale=0.1 / spread)
    s = Setup(dev, "f32", [100], [2], 2, 1, 64, 16)
    s.q[0] = 0.0
    s.q[1, 0, 1:] *= np.float32(2.0 ** -20)  # one large element, the others small
    s.check(hip)


@pytest.mark.parametrize("elem", ELEMS)
def test_hidden_places_do_not_count(hip, dev, elem):
    """Infinite and NaN keys and values in tokens that a row does not see: those past the length
    are NaN in every test here; here also those after a row's position and before its window."""
    s = Setup(dev, elem, [120], [40], 4, 2, 64, 16)
    kq = [kv_plain.quantize(s.k[0].astype(np.float32)), kv_plain.quantize(s.v[0].astype(np.float32))]
    before = s.run(hip, window=30)
    for bits in (0x7C00, 0xFC00, 0x7E00):
        for token in (20, 110):
            spoilt = [(p[0].copy(), p[1].copy()) for p in kq]
            for p in spoilt:
                p[0].view(np.uint16)[token] = bits
            s._put(s.cache, s.slots, *spoilt)
            got = s.run(hip, window=30)
            p = np.arange(80, 120)
            blind = (p < token) | (p - 30 >= token)
            assert blind.any()
            assert torch.equal(got[torch.from_numpy(blind)], before[torch.from_numpy(blind)])


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_that_are_not_finite(hip, dev, bad):
    s = Setup(dev, "f32", [90], [6], 4, 2, 64, 16)
    fine = wide(s.run(hip))
    s.q[2, 1, 7] = bad
    got = wide(s.run(hip))
    assert np.isnan(got[2, 1]).all()
    rest = np.ones((6, 4), bool)
    rest[2, 1] = False
    assert np.array_equal(got[rest], fine[rest])


def test_pages_that_are_missing(hip, dev):
    """A negative page, or one past the cache, holds no token; a row that sees only such is zero."""
    s = Setup(dev, "f32", [100, 40], [1, 1], 4, 2, 64, 16)
    table = s.table.copy()
    table[0, 2], table[0, 4], table[1, :3] = -1, s.pages, -1
    out = wide(s.run(hip, table=table))
    t = np.arange(100)
    there = ~np.isin(t // 16, (2, 4))
    want = kv_plain.attend(s.q[:1], s.k[0][there], s.v[0][there], 10 ** 6, 0.125, True, 0)
    assert (np.abs(out[:1] - want) <= s.tolerance(want)).all()
    assert (out[1] == 0.0).all()


def test_strides_and_rows_left_alone(hip, dev):
    """Queries as columns of a fused projection, an output with gaps, tokens past the last row."""
    for elem in ELEMS:
        s = Setup(dev, elem, [70, 300], [3, 1], 6, 2, 64, 16)
        plain = s.run(hip)
        rows = torch.zeros(s.tokens + 2, 11, 65, dtype=TORCH[elem], device=dev)
        rows[:s.tokens, 1:7, :64] = dev_rows(s.q, elem, dev)
        out = torch.full((s.tokens + 2, 6, 71), 5.0, dtype=TORCH[elem], device=dev)
        s.run(hip, q=rows[:, 1:7], out=out, tokens=s.tokens + 2)
        assert torch.equal(out[:s.tokens, :, :64], plain)
        out[:s.tokens, :, :64] = 5.0
        assert bool((out == 5.0).all())


def test_bounds_cut(hip, dev):
    """max_added and max_length that are smaller than the requests: what is past them is neither
    written nor read."""
    s = Setup(dev, "f32", [200], [50], 4, 2, 64, 16)
    whole = s.run(hip)
    cut = s.run(hip, max_added=20)
    assert torch.equal(cut[:20], whole[:20]) and bool((cut[20:] == 3.0).all())
    short = wide(s.run(hip, max_length=160))
    assert np.abs(short[:10] - wide(whole)[:10]).max() < 1e-5  # positions 150 .. 159 see no more
    want = kv_plain.attend(s.q[10:], s.k[0][:160], s.v[0][:160], 160, 64 ** -0.5, True, 0)
    assert (np.abs(short[10:] - want) <= s.tolerance(want)).all()


def test_streams_and_repeats(hip, dev):
    """The same bits on another stream and in every replay of a graph."""
    s = Setup(dev, "f16", [3000, 70, 900], [1, 1, 1], 8, 2, 128, 16)
    bufs, q = s.buffers(), dev_rows(s.q, s.elem, dev)
    want = s.run(hip, bufs=bufs, q=q).clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        out = s.run(hip, bufs=bufs, q=q)
    side.synchronize()
    assert torch.equal(out, want)
    out = torch.full_like(want, 3.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            s.run(hip, bufs=bufs, q=q, out=out)
    torch.cuda.synchronize()
    for _ in range(3):
        out.fill_(3.0)
        s.run(hip, bufs=bufs, q=q)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_offsets_past_32_bits(hip, dev):
    """Pages beyond 4 GiB of the cache, stored and read."""
    page, kv, dim, pages = 64, 8, 128, 60000
    size = hip.kv_q4_0_page_bytes(page, kv, dim)
    assert size * pages > 2 ** 32
    s = Setup(dev, "f32", [150], [1], 8, kv, dim, page)
    cache = torch.full((size * pages,), 0xFF, dtype=torch.uint8, device=dev)
    table = np.array([[59999, 31, 59001]], np.int32)
    t = np.arange(150)
    slots = table[0, t // page].astype(np.int64) * page + t % page
    k, v = (to_dev(x[0].astype(np.float32), dev) for x in (s.k, s.v))
    ds = to_dev(slots, dev)
    hip.kv_store_q4_0("f32", k, kv * dim, dim, v, kv * dim, dim, "half", None, None, 0, 0, ds,
                      cache, pages, page, 150, kv, dim)
    back = torch.empty(2, 150, kv, dim, device=dev)
    hip.kv_load_q4_0("f32", cache, pages, page, ds, back[0], kv * dim, dim, back[1], kv * dim, dim,
                     150, kv, dim)
    got = from_dev(back).astype(np.float64)
    s.pages, s.stride = pages, 3
    bufs = (cache, to_dev(table, dev), to_dev(s.first, dev), to_dev(s.lengths, dev))
    s.k, s.v = [got[0]], [got[1]]
    out, want = wide(s.run(hip, bufs=bufs)), s.want()
    assert (np.abs(out - want) <= s.tolerance(want)).all()
    assert np.abs(got[0] - from_dev(k)).max() < 1.0


def test_quantizer_matches_synth(hip, dev):
    """Many blocks against the quantizer that the other tests use."""
    x = synth.normal_f32(77, 512 * 2 * 256).reshape(512, 2, 256)
    cache = torch.zeros(512 * 2 * 288, dtype=torch.uint8, device=dev)
    dx = to_dev(x, dev)
    slots = torch.arange(512, device=dev)
    hip.kv_store_q4_0("f32", dx, 512, 256, dx, 512, 256, "half", None, None, 0, 0, slots, cache,
                      8, 64, 512, 2, 256)
    out = torch.empty(2, 512, 2, 256, device=dev)
    hip.kv_load_q4_0("f32", cache, 8, 64, slots, out[0], 512, 256, out[1], 512, 256, 512, 2, 256)
    want = kv_plain.values(*kv_plain.quantize(x)).astype(np.float32)
    assert np.array_equal(from_dev(out)[0], want) and np.array_equal(from_dev(out)[1], want)
