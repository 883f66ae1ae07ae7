"""The paged 4-bit cache's operators as a program that serves requests calls them through the
Python binding (tianchen-rv_amd/tcrv_hip.py): block tables and slots for the step's tokens, rotary
positions, the store of keys and values as Q4_0 blocks, and attention over the cache.

A case is a dict of plain values; `kind` says which operator:
  "tables"  block tables, slots and positions from request lengths
  "rope"    rotary positions of one tensor
  "store"   keys (rotated or as they are) and values into the cache, and the rows read back
  "attend"  attention of the requests' newest tokens over their cached tokens
  "step"    all of them in a row, over rows of one projection of queries, keys and values

listed() are the fixed cases, draw(rng) gives another of the same ranges, prepare(case, seed) makes
the device buffers, run(state) is one pass (`own` false: the plain form in torch; true: the
framework's entries), work(case) the bytes and operations that no implementation can do without,
exact(case, seed) the results in float64.

The cache, per page and kv head, for a page of P tokens and nb = dim / 32 blocks a row: P * dim / 2
bytes of keys' quants, P * nb fp16 scales, then the same for the values.  With q_b[j] byte j of a
Q4_0 block's 16 (element j low, element j + 16 high):
  keys' quants    [token][g < 4][b < nb][i < 4]                 q_b[4 g + i]
  values' quants  [token / 4][m < 16][b / 2][token % 4][b % 2]  q_b[m]
  scales          [token / 4][b < nb][token % 4]                d_b
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
ELEM = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROPE_BASE = 10000.0
MOST_TOKENS = 131072

# What a drawn case may cost at most: the listed decode over long contexts and the listed prefill.
MOST_CACHE = 2 * 131072 * 8 * 128
MOST_PRODUCTS = 4096 * 4096 * 32 * 128


def listed():
    return [
        # The smallest call: the tables of one decode step of sixty-four sequences.
        dict(name="tables_decode", kind="tables", requests=64, context=4096, added=1, page=16,
             mix=1),
        # Prompts of many requests admitted at once: ragged lengths, pages of 64.
        dict(name="tables_prompts", kind="tables", requests=301, context=900, added=700, page=64,
             mix=2),
        # Queries of seven sequences' next tokens; latency.
        dict(name="rope_decode", kind="rope", elem="bf16", layout="half", tokens=7, heads=32,
             dim=128, rot=128, span=32768, inverse=False),
        # A prompt's queries, half of each head rotated, pairs interleaved.
        dict(name="rope_prompt", kind="rope", elem="f32", layout="interleaved", tokens=4096,
             heads=32, dim=128, rot=64, span=131072, inverse=False),
        # The next tokens of sixty-four sequences into the cache, keys rotated.
        dict(name="store_decode", kind="store", elem="f16", layout="half", tokens=64, heads=8,
             dim=128, rot=128, page=16, span=8192),
        # Prompts into the cache: an odd count, fp32 as the quantized GEMMs write it.
        dict(name="store_prompt", kind="store", elem="f32", layout="half", tokens=8191, heads=8,
             dim=128, rot=128, page=64, span=16384),
        # One sequence early in its answer: latency.
        dict(name="attend_one", kind="attend", elem="f32", requests=1, context=531, added=1,
             heads=32, kv_heads=8, dim=128, page=16, causal=True, window=0, mix=3),
        # Batched decode: sixty-four sequences, contexts ragged up to 8192.
        dict(name="attend_batch", kind="attend", elem="f16", requests=64, context=8192, added=1,
             heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0, mix=4),
        # Two long documents, a token each: the largest read of a cache.
        dict(name="attend_long", kind="attend", elem="bf16", requests=2, context=131072, added=1,
             heads=32, kv_heads=8, dim=128, page=32, causal=True, window=0, mix=5),
        # Prefill: one prompt, every token against those before it; the largest product.
        dict(name="attend_prefill", kind="attend", elem="f16", requests=1, context=4096,
             added=4096, heads=32, kv_heads=8, dim=128, page=64, causal=True, window=0, mix=6),
        # Chunked prefill beside decode: ragged chunks on long contexts, a sliding window,
        # small heads, seven queries a kv head.
        dict(name="attend_chunks", kind="attend", elem="f32", requests=9, context=6000, added=300,
             heads=14, kv_heads=2, dim=64, page=48, causal=True, window=2047, mix=7),
        # A decode step of thirty-two sequences through all of them.
        dict(name="step_decode", kind="step", elem="f32", layout="half", requests=32, context=4096,
             added=1, heads=32, kv_heads=8, dim=128, rot=128, page=32, mix=8),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _fit(case):
    """Shortens a drawn case until it costs no more than the largest listed ones."""
    while True:
        pairs, cached, tokens = 0, 0, 0
        for length, added in _lengths(case):
            cached += length
            tokens += added
            pairs += added * length
        if (cached * case["kv_heads"] * case["dim"] <= MOST_CACHE
                and pairs * case["heads"] * case["dim"] <= MOST_PRODUCTS
                and cached * case["heads"] <= 1 << 24 and tokens <= 16384):
            return case
        if case["added"] > 64 and pairs * case["heads"] * case["dim"] > MOST_PRODUCTS:
            case["added"] = max(64, case["added"] * 3 // 4)
        elif case["requests"] > 1 and case["context"] < 4096:
            case["requests"] = max(1, case["requests"] * 3 // 4)
        else:
            case["context"] = max(1, case["context"] * 3 // 4)
            case["added"] = min(case["added"], case["context"])


def draw(rng):
    kind = rng.choice(("tables", "rope", "store", "attend", "attend", "attend", "attend", "step"))
    page = rng.choice((16, 16, 32, 48, 64, 128))
    elem = rng.choice(("f32", "f16", "bf16"))
    heads, kv_heads = rng.choice(((32, 8), (32, 32), (8, 1), (28, 4), (40, 8), (14, 2), (64, 8)))
    dim = rng.choice((64, 128, 128, 128, 192, 256))
    layout = rng.choice(("half", "interleaved"))
    rot = rng.choice((dim, dim, dim // 2))
    mix = rng.randrange(1 << 20)
    if kind == "tables":
        context = _log_uniform(rng, 1, 16384)
        requests = _log_uniform(rng, 1, 1024)
        added = 1 if rng.random() < 0.5 else _log_uniform(rng, 1, 2048)
        return dict(kind=kind, requests=requests, context=max(context, added),
                    added=min(added, MOST_TOKENS // requests), page=page, mix=mix)
    if kind == "rope":
        tokens = min(_log_uniform(rng, 1, 8192), 4096 * 32 * 128 // (heads * dim))
        return dict(kind=kind, elem=elem, layout=layout, tokens=tokens, heads=heads, dim=dim,
                    rot=rot, span=_log_uniform(rng, 4096, 131072), inverse=rng.random() < 0.3)
    if kind == "store":
        tokens = min(_log_uniform(rng, 1, 8192), 8191 * 8 * 128 // (kv_heads * dim))
        return dict(kind=kind, elem=elem, layout=layout, tokens=tokens, heads=kv_heads, dim=dim,
                    rot=rng.choice((rot, rot, 0)), page=page, span=_log_uniform(rng, 4096, 65536))
    case = dict(kind=kind, elem=elem, requests=_log_uniform(rng, 1, 128),
                context=_log_uniform(rng, 16, 131072), added=1, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, mix=mix)
    if kind == "step":
        case.update(layout=layout, rot=rot, added=rng.choice((1, 1, 4)))
        case["context"] = min(case["context"], 16384)
        return _fit(case)
    case.update(causal=rng.random() < 0.85, window=0)
    shape = rng.choice(("decode", "decode", "few", "chunk", "prefill"))
    if shape == "few":
        case["added"] = rng.randint(2, 8)
    elif shape == "chunk":
        case.update(added=_log_uniform(rng, 16, 512), requests=_log_uniform(rng, 1, 16))
        case["context"] = min(case["context"], 32768)
    elif shape == "prefill":
        case.update(requests=rng.randint(1, 4), context=min(case["context"], 8192))
        case["added"] = case["context"]
    case["added"] = min(case["added"], case["context"])
    if rng.random() < 0.25:
        case["window"] = _log_uniform(rng, 16, 4096)
    return _fit(case)


def _lengths(case):
    """[(length, added)] of the requests: tokens cached with the newest, and the newest.  The first
    request has the most of both; of many, one has no new token."""
    rng = random.Random(case["mix"])
    got = [(case["context"], case["added"])]
    for r in range(1, case["requests"]):
        added = case["added"] if case["added"] <= 1 else rng.randint(1, case["added"])
        length = max(added, rng.randint(max(1, case["context"] // 8), case["context"]))
        got.append((length, 0 if r == 5 else added))
    return got


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _channels(gen, heads, dim):
    """The spread of a projection's channels: a few of them ten times the others."""
    spread = 0.5 + torch.rand(heads, dim, generator=gen, device=DEV)
    loud = torch.rand(heads, dim, generator=gen, device=DEV) < 0.03
    return torch.where(loud, spread * 10.0, spread)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _rope_table(rot, rows):
    """float32 [rows, rot / 2, 2]: cosine and sine of position * base^(-2 i / rot)."""
    i = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    angle = (torch.arange(rows, device=DEV, dtype=torch.float64)[:, None]
             * ROPE_BASE ** (-2.0 * i / rot))
    return torch.stack((angle.cos(), angle.sin()), dim=-1).float().contiguous()


def _quantize(x):
    """float32 [..., 32] -> Q4_0: (fp16 scales [...], uint8 quants [..., 32]).  The scale is the
    element of largest magnitude (the first of several) over -8."""
    mag = x.abs()
    place = torch.arange(32, device=x.device)
    first = torch.where(mag == mag.amax(-1, keepdim=True), place, 32).amin(-1, keepdim=True)
    d = x.gather(-1, first.clamp(max=31)) / -8.0
    inv = torch.where(d == 0, torch.zeros_like(d), torch.ones_like(d) / d)
    q = (x * inv + 8.5).floor().clamp(0, 15).to(torch.uint8)
    return d[..., 0].half(), q


def _page_bytes(page, heads, dim):
    return heads * page * dim * 9 // 8


def _views(cache, page, heads, dim):
    """The parts of a cache (uint8) as views: quants and scales of keys, then of values."""
    nb, quants, scales = dim // 32, page * dim // 2, page * dim // 16
    rows = cache.view(-1, heads, page * dim * 9 // 8)
    at, half, n = quants + scales, torch.float16, rows.shape[0]
    return (rows[..., :quants].view(n, heads, page, 4, nb, 4),
            rows[..., quants:at].view(half).view(n, heads, page // 4, nb, 4),
            rows[..., at:at + quants].view(n, heads, page // 4, 16, nb // 2, 4, 2),
            rows[..., at + quants:].view(half).view(n, heads, page // 4, nb, 4))


def _place(cache, page, heads, dim, slots, k, v):
    """Writes the quantized rows ((scales [tokens, heads, nb], quants [tokens, heads, nb, 32]) of
    keys and values) at their slots."""
    nb = dim // 32
    kq, ks, vq, vs = _views(cache, page, heads, dim)
    at, off = slots // page, slots % page
    group, lane = off // 4, off % 4
    qs = k[1][..., :16] | (k[1][..., 16:] << 4)
    kq[at, :, off] = qs.view(-1, heads, nb, 4, 4).transpose(2, 3)
    ks[at, :, group, :, lane] = k[0]
    qs = v[1][..., :16] | (v[1][..., 16:] << 4)
    vq[at, :, group, :, :, lane] = qs.view(-1, heads, nb // 2, 2, 16).permute(0, 1, 4, 2, 3)
    vs[at, :, group, :, lane] = v[0]


def _values(scales, quants):
    """Q4_0 -> float32 [..., nb * 32] from scales [..., nb] and the 16 bytes of a block
    [..., nb, 16]."""
    q = torch.cat((quants & 15, quants >> 4), dim=-1).float() - 8.0
    return (q * scales.float()[..., None]).flatten(-2)


def _read(cache, page, heads, dim, slots):
    """(keys, values) float32 [tokens, heads, dim] at their slots."""
    nb = dim // 32
    kq, ks, vq, vs = _views(cache, page, heads, dim)
    at, off = slots // page, slots % page
    group, lane = off // 4, off % 4
    n = slots.shape[0]
    k = kq[at, :, off].transpose(2, 3).reshape(n, heads, nb, 16)
    v = vq[at, :, group, :, :, lane].permute(0, 1, 3, 4, 2).reshape(n, heads, nb, 16)
    return _values(ks[at, :, group, :, lane], k), _values(vs[at, :, group, :, lane], v)


def _tables_inputs(case, seed):
    """Lengths before the step, tokens added, the pages of the cached tokens and free ones."""
    rows = _lengths(case)
    page = case["page"]
    before = [length - added for length, added in rows]
    held = [-(-c // page) for c in before]
    new = [-(-length // page) - h for (length, _), h in zip(rows, held)]
    width = max(-(-length // page) for length, _ in rows)
    pages = sum(held) + sum(new) + 7
    shuffled = torch.randperm(pages, generator=_generator(seed), device=DEV).to(torch.int32)
    width_at = torch.arange(width, device=DEV)
    start = torch.cumsum(_ints([0] + held[:-1]).long(), 0)
    have = width_at[None] < _ints(held)[:, None]
    block_table = torch.where(have, shuffled[(start[:, None] + width_at).clamp(max=pages - 1)],
                              torch.full((), -1, dtype=torch.int32, device=DEV)).contiguous()
    return dict(context=_ints(before), added=_ints([added for _, added in rows]),
                block_table=block_table, free=shuffled[sum(held):].contiguous(), pages=pages,
                width=width, tokens=sum(added for _, added in rows),
                # what a scheduler knows of the lengths without reading them back
                most_added=case["added"], most_context=case["context"])


def _cached(case, gen, r, length):
    """Request r's quantized keys and values, [length, kv_heads, nb(, 32)]."""
    kv, nb = case["kv_heads"], case["dim"] // 32
    spread = _channels(gen, kv, case["dim"])
    k = _quantize((_normal(gen, length, kv, case["dim"]) * spread).view(length, kv, nb, 32))
    v = _quantize(_normal(gen, length, kv, case["dim"]).view(length, kv, nb, 32))
    return k, v


def _queries(case, seed, tokens):
    """Rows whose scores spread over a few units, as a trained head's do."""
    gen = _generator(seed * 7919 + 1)
    return (_normal(gen, tokens, case["heads"], case["dim"]) * 0.5).to(ELEM[case["elem"]])


def _fused_rows(case, seed, tokens):
    """The rows of one projection: queries, keys and values side by side."""
    gen = _generator(seed * 7919 + 2)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    x = _normal(gen, tokens, heads + 2 * kv, dim)
    x[:, :heads] *= 0.5
    return x.to(ELEM[case["elem"]])


def prepare(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return dict(case, **_tables_inputs(case, seed))
    if kind in ("rope", "store"):
        gen = _generator(seed)
        tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
        state = dict(case, positions=torch.randint(0, case["span"], (tokens,), generator=gen,
                                                   device=DEV, dtype=torch.int32))
        state["table"] = _rope_table(case["rot"], case["span"]) if case["rot"] else None
        if kind == "rope":
            state["x"] = _normal(gen, tokens, heads, dim).to(ELEM[case["elem"]])
            return state
        state["k"] = (_normal(gen, tokens, heads, dim)
                      * _channels(gen, heads, dim)).to(ELEM[case["elem"]])
        state["v"] = _normal(gen, tokens, heads, dim).to(ELEM[case["elem"]])
        pages = -(-tokens // case["page"]) + 3
        order = torch.randperm(pages, generator=gen, device=DEV)
        at = torch.arange(tokens, device=DEV)
        state["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        state["pages"] = pages
        state["cache"] = torch.full((pages * _page_bytes(case["page"], heads, dim),), 255,
                                    dtype=torch.uint8, device=DEV)
        return state
    # The cache as the steps before have left it: what no token was stored in yet is 0xff.
    rows = _lengths(case)
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    state = dict(case, **_tables_inputs(case, seed))
    state["cache"] = torch.full((state["pages"] * _page_bytes(page, kv, dim),), 255,
                                dtype=torch.uint8, device=DEV)
    filled = state if kind == "step" else dict(state, **_tables(state))
    gen = _generator(seed * 7919)
    for r, (length, added) in enumerate(rows):
        k, v = _cached(case, gen, r, length)
        n = length - added if kind == "step" else length
        at = torch.arange(n, device=DEV)
        slots = filled["block_table"][r].long()[at // page] * page + at % page
        _place(state["cache"], page, kv, dim, slots, [x[:n] for x in k], [x[:n] for x in v])
    if kind == "step":
        state["rows"] = _fused_rows(case, seed, state["tokens"])
        state["table"] = _rope_table(case["rot"], case["context"])
        return state
    state.update({name: filled[name] for name in ("block_table", "first", "length")})
    state["q"] = _queries(case, seed, state["tokens"])
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _tables(s):
    """block_table with the new tokens' pages, first, length, positions, slots, taken."""
    page, context, added = s["page"], s["context"].long(), s["added"].long()
    length = context + added
    held, need = -(-context // page), -(-length // page)
    end = torch.cumsum(added, 0)
    took = torch.cumsum(need - held, 0)
    column = torch.arange(s["width"], device=DEV)[None]
    new = (column >= held[:, None]) & (column < need[:, None])
    source = (took - need)[:, None] + column
    table = torch.where(new, s["free"].long()[source.clamp(0, s["free"].shape[0] - 1)],
                        s["block_table"].long())
    i = torch.arange(s["tokens"], device=DEV)
    r = torch.searchsorted(end, i, right=True)
    position = context[r] + i - (end - added)[r]
    slots = table[r, position // page] * page + position % page
    first = torch.cat((torch.zeros_like(end[:1]), end))
    return dict(block_table=table.int(), first=first.int(), length=length.int(),
                positions=position.int(), slots=slots, taken=took[-1:].int())


def _rope(x, positions, table, rot, layout, inverse=False):
    """float32 result of rotating the first `rot` elements of [tokens, heads, dim]."""
    x = x.float()
    turn = table[positions.long()][:, None]
    c, sn = turn[..., 0], -turn[..., 1] if inverse else turn[..., 1]
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat((a * c - b * sn, a * sn + b * c, x[..., rot:]), dim=-1)
    a, b = x[..., :rot:2], x[..., 1:rot:2]
    turned = torch.stack((a * c - b * sn, a * sn + b * c), dim=-1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), dim=-1)


def _store(s, k, v, positions, slots, heads):
    nb, dim = s["dim"] // 32, s["dim"]
    k = _rope(k, positions, s["table"], s["rot"], s["layout"]) if s["rot"] else k.float()
    _place(s["cache"], s["page"], heads, dim, slots, _quantize(k.reshape(-1, heads, nb, 32)),
           _quantize(v.float().reshape(-1, heads, nb, 32)))


def _attend(s, q, block_table, first, length, causal, window):
    """float32 [tokens, heads, dim]: softmax(q k' / sqrt(dim)) v over each request's tokens."""
    heads, kv, dim, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    n, most = block_table.shape[0], s["most_added"]
    slots = (block_table.clamp(min=0).long()[..., None] * page
             + torch.arange(page, device=DEV)).reshape(-1)
    k, v = _read(s["cache"], page, kv, dim, slots)
    k, v = (x.view(n, -1, kv, dim).transpose(1, 2) for x in (k, v))
    t = torch.arange(k.shape[2], device=DEV)
    v = torch.where((t < length[:, None])[:, None, :, None], v, torch.zeros_like(v))
    added = first[1:] - first[:-1]
    i = torch.arange(most, device=DEV)
    token = (first[:-1, None] + i).clamp(max=q.shape[0] - 1).long()
    rows = q.float()[token].view(n, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(rows.reshape(n, kv, -1, dim) * dim ** -0.5, k.transpose(2, 3))
    at = (length - added)[:, None] + i
    seen = (t < length[:, None])[:, None].expand(-1, most, -1)
    if causal:
        seen = seen & (t <= at[..., None])
    if window:
        seen = seen & (t > at[..., None] - window)
    scores = scores.view(n, kv, -1, most, t.shape[0])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, kv, -1, t.shape[0]), v).view(n, kv, -1, most, dim)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 3, 1, 2, 4).reshape(n, most, heads, dim)[i < added[:, None]]


def _plain(s):
    kind = s["kind"]
    if kind == "tables":
        return _tables(s)
    if kind == "rope":
        return _rope(s["x"], s["positions"], s["table"], s["rot"], s["layout"],
                     s["inverse"]).to(ELEM[s["elem"]])
    if kind == "store":
        _store(s, s["k"], s["v"], s["positions"], s["slots"], s["heads"])
        k, v = _read(s["cache"], s["page"], s["heads"], s["dim"], s["slots"])
        return {"k": k, "v": v}
    if kind == "attend":
        return _attend(s, s["q"], s["block_table"], s["first"], s["length"], s["causal"],
                       s["window"]).to(ELEM[s["elem"]])
    t = _tables(s)
    heads, kv = s["heads"], s["kv_heads"]
    q, k, v = s["rows"].split((heads, kv, kv), dim=1)
    q = _rope(q, t["positions"], s["table"], s["rot"], s["layout"]).to(ELEM[s["elem"]])
    _store(s, k, v, t["positions"], t["slots"], kv)
    out = _attend(s, q, t["block_table"], t["first"], t["length"], True, 0)
    return dict(t, out=out.to(ELEM[s["elem"]]))


# ---------------------------------------------------------------------------
# The framework's entries
# ---------------------------------------------------------------------------

def _binding():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "tianchen-rv_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tcrv_hip
    return tcrv_hip


def _own_tables(hip, s):
    n, tokens = s["context"].shape[0], s["tokens"]
    out = s.setdefault("made", dict(
        first=torch.empty(n + 1, dtype=torch.int32, device=DEV),
        length=torch.empty(n, dtype=torch.int32, device=DEV),
        positions=torch.empty(tokens, dtype=torch.int32, device=DEV),
        slots=torch.empty(tokens, dtype=torch.int64, device=DEV),
        taken=torch.empty(1, dtype=torch.int32, device=DEV)))
    hip.kv_tables(s["context"], s["added"], n, s["page"], s["free"], s["free"].shape[0],
                  s["block_table"], s["width"], out["first"], out["length"], out["positions"],
                  out["slots"], tokens, out["taken"])
    return dict(out, block_table=s["block_table"])


def _own_store(hip, s, k, v, positions, slots, heads):
    rows = s["table"].shape[0] if s["rot"] else 0
    hip.kv_store_q4_0(s["elem"], k, k.stride(0), k.stride(1), v, v.stride(0), v.stride(1),
                      s["layout"], positions, s["table"], rows, s["rot"], slots, s["cache"],
                      s["pages"], s["page"], k.shape[0], heads, s["dim"])


def _own_attend(hip, s, q, block_table, first, length, causal, window):
    n, heads, kv, dim = block_table.shape[0], s["heads"], s["kv_heads"], s["dim"]
    if "out" not in s:
        need = hip.attn_q4_0_workspace_bytes(s["elem"], n, q.shape[0], s["most_added"],
                                             s["most_context"], heads, kv, dim)
        s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
        s["out"] = torch.empty_like(q, memory_format=torch.contiguous_format)
    out = s["out"]
    hip.attn_q4_0(s["elem"], q, q.stride(0), q.stride(1), s["cache"], s["pages"], s["page"],
                  block_table, s["width"], first, length, n, q.shape[0], s["most_added"],
                  s["most_context"], heads, kv, dim, dim ** -0.5, causal, window, out,
                  out.stride(0), out.stride(1), s["workspace"], s["workspace"].numel())
    return out


def _own_rope(hip, s, x, positions, inverse=False):
    y = s.setdefault("turned", torch.empty(x.shape, dtype=x.dtype, device=DEV))
    hip.rope(s["elem"], s["layout"], x, x.stride(0), x.stride(1), y, y.stride(0), y.stride(1),
             positions, s["table"], s["table"].shape[0], x.shape[0], x.shape[1], s["dim"],
             s["rot"], inverse)
    return y


def _framework(s):
    hip, kind = _binding(), s["kind"]
    if kind == "tables":
        return _own_tables(hip, s)
    if kind == "rope":
        return _own_rope(hip, s, s["x"], s["positions"], s["inverse"])
    if kind == "store":
        _own_store(hip, s, s["k"], s["v"], s["positions"], s["slots"], s["heads"])
        shape = s["tokens"], s["heads"], s["dim"]
        k, v = s.setdefault("read", (torch.empty(shape, device=DEV),
                                     torch.empty(shape, device=DEV)))
        hip.kv_load_q4_0("f32", s["cache"], s["pages"], s["page"], s["slots"], k, k.stride(0),
                         k.stride(1), v, v.stride(0), v.stride(1), s["tokens"], s["heads"],
                         s["dim"])
        return {"k": k, "v": v}
    if kind == "attend":
        return _own_attend(hip, s, s["q"], s["block_table"], s["first"], s["length"], s["causal"],
                           s["window"])
    t = _own_tables(hip, s)
    heads, kv = s["heads"], s["kv_heads"]
    q, k, v = s["rows"].split((heads, kv, kv), dim=1)
    q = _own_rope(hip, s, q, t["positions"])
    _own_store(hip, s, k, v, t["positions"], t["slots"], kv)
    return dict(t, out=_own_attend(hip, s, q, t["block_table"], t["first"], t["length"], True, 0))


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# The least work, and the results in float64
# ---------------------------------------------------------------------------

def _seen(length, added, causal, window):
    """Pairs of a new token and a cached one that it sees, and the cached tokens that any sees."""
    pairs, low = 0, length
    for at in range(length - added, length):
        end = at + 1 if causal else length
        begin = max(0, at - window + 1) if window else 0
        pairs += max(0, end - begin)
        low = min(low, begin)
    return pairs, (length - low if added else 0)


def work(case):
    kind = case["kind"]
    if kind == "rope":
        size = {"f32": 4}.get(case["elem"], 2)
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * size + case["tokens"] * (4 + case["rot"] * 4),
                "flops": n * case["rot"] * 3}
    if kind == "store":
        size = {"f32": 4}.get(case["elem"], 2)
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * size + 2 * n * 9 // 16 + 2 * n * 4
                + case["tokens"] * (12 + case["rot"] * 4), "flops": 2 * n * 3}
    rows, page = _lengths(case), case["page"]
    tokens = sum(added for _, added in rows)
    new = sum(-(-length // page) + -(-(added - length) // page) for length, added in rows)
    tables = len(rows) * 20 + new * 8 + tokens * 12
    if kind == "tables":
        return {"bytes": tables, "flops": 2 * tokens}
    size = {"f32": 4}.get(case["elem"], 2)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    pairs = cached = 0
    for length, added in rows:
        p, c = _seen(length, added, case.get("causal", True), case.get("window", 0))
        pairs, cached = pairs + p, cached + c
    got = {"bytes": cached * kv * dim * 9 // 8 + 2 * tokens * heads * dim * size,
           "flops": 4 * pairs * heads * dim}
    if kind == "step":
        got["bytes"] += tables + tokens * (kv * dim * (16 * size + 9) // 8 + 4 * case["rot"])
    return got


def _exact_attention(case, q, k, v, length, added, causal, window):
    """One request's rows in float64: q [added, heads, dim], k and v [length, kv_heads, dim]."""
    out = torch.empty(added, case["heads"], case["dim"], dtype=torch.float64, device=DEV)
    at = torch.arange(length - added, length, device=DEV)[:, None]
    t = torch.arange(length, device=DEV)[None]
    hidden = torch.zeros(added, length, dtype=torch.bool, device=DEV)
    if causal:
        hidden |= t > at
    if window:
        hidden |= t <= at - window
    share = case["heads"] // case["kv_heads"]
    for h in range(case["heads"]):
        z = (q[:, h] @ k[:, h // share].t()) / math.sqrt(case["dim"])
        out[:, h] = torch.softmax(z.masked_fill(hidden, -math.inf), dim=1) @ v[:, h // share]
    return out


def _wide(part):
    return ((part[1].double() - 8.0) * part[0].double()[..., None]).flatten(-2)


def _turned(x, positions, rot, layout, inverse=False):
    """Pairs as complex numbers times e^(i angle), in float64."""
    x = x.double()
    i = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    angle = positions.double()[:, None, None] * ROPE_BASE ** (-2.0 * i / rot)
    turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle)
    out = x.clone()
    if layout == "half":
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
        out[..., :rot // 2], out[..., rot // 2:rot] = z.real, z.imag
    else:
        z = torch.complex(x[..., :rot:2], x[..., 1:rot:2]) * turn
        out[..., :rot:2], out[..., 1:rot:2] = z.real, z.imag
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "rope":
        s = prepare(case, seed)
        return _turned(s["x"], s["positions"], s["rot"], s["layout"], s["inverse"])
    if kind in ("tables", "store"):  # whole numbers, and values rounded to 4 bits, have no other
        return None
    rows = _lengths(case)
    tokens = sum(added for _, added in rows)
    gen = _generator(seed * 7919)
    fused = _fused_rows(case, seed, tokens) if kind == "step" else None
    q = fused[:, :case["heads"]] if kind == "step" else _queries(case, seed, tokens)
    got, at = [], 0
    for r, (length, added) in enumerate(rows):
        k, v = (_wide(part) for part in _cached(case, gen, r, length))
        mine = q[at:at + added]
        if kind == "step":
            heads, kv, nb = case["heads"], case["kv_heads"], case["dim"] // 32
            where = torch.arange(length - added, length, device=DEV)
            mine = _turned(mine, where, case["rot"], case["layout"]).to(q.dtype)
            new = _turned(fused[at:at + added, heads:heads + kv], where, case["rot"],
                          case["layout"]).float()
            k[length - added:] = _wide(_quantize(new.reshape(added, kv, nb, 32)))
            new = fused[at:at + added, heads + kv:].float()
            v[length - added:] = _wide(_quantize(new.reshape(added, kv, nb, 32)))
        got.append(_exact_attention(case, mine.double(), k, v, length, added,
                                    case.get("causal", True), case.get("window", 0)))
        at += added
    out = torch.cat(got)
    if kind == "attend":
        return out
    return dict.fromkeys(("block_table", "first", "length", "positions", "slots", "taken"),
                         None) | {"out": out}
