"""Plain forms of the paged Q4_0 cache's operators for the tests: numpy, the formulas of
include/tcrv_hip.h written out, attention in float64."""
import numpy as np

import synth

I32_MAX = 2 ** 31 - 1


def round_to(x, elem):
    """float32 values of `x` rounded to the element type (nearest even)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if elem == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    if elem == "bf16":
        u = x.view(np.uint32).astype(np.uint64)
        up = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32)
        return np.where(np.isnan(x), np.float32(np.nan), up.view(np.float32))
    return x


def tables(context, added, page_size, free, block_table, max_tokens):
    """The outputs of tcrv_hip_kv_tables, request by request."""
    table = block_table.copy()
    stride = table.shape[1]
    first, length, positions, slots, taken = [0], [], [], [], 0
    for r, (c, a) in enumerate(zip(context, added)):
        c, a = max(int(c), 0), max(int(a), 0)
        held, need = min(-(-c // page_size), stride), min(-(-(c + a) // page_size), stride)
        for column in range(held, need):
            table[r, column] = max(int(free[taken]), -1) if taken < len(free) else -1
            taken += 1
        for p in range(c, c + a):
            column = p // page_size
            page = int(table[r, column]) if column < stride else -1
            positions.append(p)
            slots.append(page * page_size + p % page_size if page >= 0 else -1)
        first.append(len(positions))
        length.append(c + a)
    pad = max(0, max_tokens - len(positions))
    return dict(block_table=table, first=np.array(first, np.int32),
                length=np.array(length, np.int32),
                positions=np.array(positions + [-1] * pad, np.int32)[:max_tokens],
                slots=np.array(slots + [-1] * pad, np.int64)[:max_tokens],
                taken=np.array([taken], np.int32))


def rope_angles(n_dims, positions, base, scaling="none", factor=1.0, trained=4096.0,
                beta_fast=32.0, beta_slow=1.0, divisors=None):
    """(angles float64 [positions, n_dims / 2], amplitude)."""
    n, amplitude = n_dims, 1.0
    i = np.arange(n // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (n / (n - 2.0))
    f = base ** (-2.0 * i / n)
    if divisors is not None:
        f = f / divisors.astype(np.float64)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def place(beta):
            return n * np.log(trained / (beta * 2.0 * np.pi)) / (2.0 * np.log(base))
        low = max(np.floor(place(beta_fast)), 0.0)
        high = min(np.ceil(place(beta_slow)), n - 1.0)
        r = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
        f = f * (1.0 - r) + f / factor * r
        amplitude = 0.1 * np.log(factor) + 1.0
    return np.asarray(positions, np.float64)[:, None] * f, amplitude


def rope(x, positions, table, n_dims, layout, inverse=False):
    """float32 [tokens, heads, dim], every product and sum rounded on its own."""
    y = x.astype(np.float32).copy()
    half = n_dims // 2
    a, b = ((slice(0, half), slice(half, n_dims)) if layout == "half" else
            (slice(0, n_dims, 2), slice(1, n_dims, 2)))
    for t, p in enumerate(positions):
        if 0 <= p < table.shape[0] and n_dims:
            c, s = table[p, :, 0], table[p, :, 1] * np.float32(-1.0 if inverse else 1.0)
            xa, xb = x[t][:, a].astype(np.float32), x[t][:, b].astype(np.float32)
            y[t][:, a] = xa * c - xb * s
            y[t][:, b] = xa * s + xb * c
    return y


def quantize(x):
    """float32 [tokens, heads, dim] -> (scales float16 [.., nb], bytes uint8 [.., nb, 16])."""
    blocks = synth.quantize_q4_0(x).reshape(*x.shape[:2], x.shape[2] // 32, 18)
    return blocks[..., :2].copy().view(np.float16)[..., 0], blocks[..., 2:].copy()


def values(scales, quants):
    """float64 [tokens, heads, dim] that the blocks stand for."""
    q = np.concatenate([quants & 15, quants >> 4], axis=-1).astype(np.float64) - 8.0
    with np.errstate(invalid="ignore"):
        v = q * scales.astype(np.float64)[..., None]
    return v.reshape(*v.shape[:-2], v.shape[-2] * 32)


class Cache:
    """A cache's bytes, written one token at a time by the layout's formula."""

    def __init__(self, pages, page_size, heads, dim, fill=0xFF):
        self.page_size, self.heads, self.dim, self.nb = page_size, heads, dim, dim // 32
        self.quants, self.scales = page_size * dim // 2, page_size * dim // 16
        self.pages = pages
        self.bytes = np.full((pages, heads, 2 * (self.quants + self.scales)), fill, np.uint8)

    def _scale_at(self, t):
        return [((t // 4) * self.nb + b) * 8 + (t % 4) * 2 for b in range(self.nb)]

    def put(self, slot, head, which, scales, quants):
        page, t = divmod(int(slot), self.page_size)
        at = self.bytes[page, head]
        nb, values_at = self.nb, self.quants + self.scales
        if which == "k":
            for g in range(4):
                for b in range(nb):
                    o = (t * 4 + g) * nb * 4 + b * 4
                    at[o:o + 4] = quants[b, 4 * g:4 * g + 4]
        else:
            for m in range(16):
                for b in range(nb):
                    o = (((t // 4) * 16 + m) * (nb // 2) + b // 2) * 8 + (t % 4) * 2 + b % 2
                    at[values_at + o] = quants[b, m]
        base = self.quants if which == "k" else values_at + self.quants
        for b, o in enumerate(self._scale_at(t)):
            at[base + o:base + o + 2] = scales[b:b + 1].view(np.uint8)

    def store(self, slots, k, v):
        """k, v: (scales, bytes) of quantize()."""
        for i, slot in enumerate(slots):
            if 0 <= slot < self.pages * self.page_size:
                for h in range(self.heads):
                    self.put(slot, h, "k", k[0][i, h], k[1][i, h])
                    self.put(slot, h, "v", v[0][i, h], v[1][i, h])


def attend(q, keys, vals, position0, scale, causal, window):
    """One request in float64: q [added, heads, dim] at positions position0 .., keys and vals
    [length, kv_heads, dim]."""
    added, heads, dim = q.shape
    length, kv, _ = keys.shape
    share = heads // kv
    t = np.arange(length)
    out = np.zeros((added, heads, dim))
    for i in range(added):
        p = position0 + i
        seen = np.ones(length, bool)
        if causal:
            seen &= t <= p
        if window:
            seen &= t > p - window
        if not seen.any():
            continue
        for h in range(heads):
            z = scale * (keys[seen, h // share] @ q[i, h].astype(np.float64))
            w = np.exp(z - z.max())
            out[i, h] = w @ vals[seen, h // share] / w.sum()
    return out
