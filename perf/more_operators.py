"""The operators between a step's quantized products, and those of drafted tokens, as a program that
serves requests calls them through the Python binding (tianchen-rv_amd/tcrv_hip.py).

A case is a dict of plain values; `kind` says which operator:
  "norm"    the residual's addition and the root-mean-square norm, in an element type or as Q8_0 blocks
  "gated"   the first half of a gated feed-forward: both Q4_0 projections of Q8_0 rows, the activation
            of the one and its product with the other, in an element type or as Q8_0 blocks
  "tree"    what each drafted token of a tree sees of the others, and its position
  "attend"  attention of the drafted tokens over the paged 4-bit cache, each token seeing its request's
            cached tokens and its own ancestors
  "keep"    the tokens of the tree that were accepted moved to the places that follow the cached ones

listed() are the fixed cases, draw(rng) gives another of the same ranges, prepare(case, seed) makes
the device buffers, run(state) is one pass (`own` false: the plain form in torch; true: the
framework's entries), work(case) the bytes and operations that no implementation can do without,
exact(case, seed) the results in float64.

Q8_0 blocks are returned as the values they stand for.  Those of "gated" come as float16: a value next
to the border of two quants falls to either side by the last bit of a sum, whatever computes it, so that
the blocks have no more than their 8 bits in common.  Those of "norm" are the same whatever computes them:
the mean is a sum in 64 bits, its root rounded once, and what follows are single operations in 32 bits.

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
EPS = 1e-5

# What a drawn case may cost at most: the listed prompts and trees.
MOST_NORM = 4096 * 4096
MOST_PRODUCTS = 2 * 14336 * 4096 * 2048
MOST_WEIGHTS = 2 * 14336 * 4096
MOST_CACHED = 64 * 4096
MOST_SCORES = 64 * 4096 * 32 * 8


def listed():
    return [
        # The next token of one sequence, between two layers: latency.
        dict(name="norm_decode", kind="norm", elem="f32", tokens=1, dim=4096, out="elem"),
        # A prompt's rows on their way into the next quantized product.
        dict(name="norm_prompt", kind="norm", elem="f16", tokens=4096, dim=4096, out="q8_0"),
        # The next token of one sequence: two matrices read once.
        dict(name="gated_decode", kind="gated", elem="f32", act="silu", tokens=1, dim=4096,
             wide=14336, out="elem"),
        # Batched decode: twenty-nine sequences, tanh form of the Gaussian unit.
        dict(name="gated_batch", kind="gated", elem="f16", act="gelu_tanh", tokens=29, dim=4096,
             wide=11008, out="elem"),
        # A prompt, its rows on their way into the down projection; the largest product.
        dict(name="gated_prompt", kind="gated", elem="f32", act="silu", tokens=2048, dim=4096,
             wide=14336, out="q8_0"),
        # The trees of a few sequences.
        dict(name="tree_few", kind="tree", requests=4, nodes=64, context=4096, mix=1),
        # Many sequences, small ragged trees.
        dict(name="tree_many", kind="tree", requests=301, nodes=17, context=4096, mix=2),
        # One sequence early in its answer, a few drafted tokens: latency.
        dict(name="attend_one", kind="attend", elem="f32", requests=1, context=531, nodes=7,
             heads=32, kv_heads=8, dim=128, page=16, window=0, mix=3),
        # Batched: sixty-four sequences, contexts ragged up to 4096, eight drafted tokens each.
        dict(name="attend_batch", kind="attend", elem="f16", requests=64, context=4096, nodes=8,
             heads=32, kv_heads=8, dim=128, page=64, window=0, mix=4),
        # Large trees of a few sequences on long contexts.
        dict(name="attend_wide", kind="attend", elem="bf16", requests=6, context=8192, nodes=64,
             heads=32, kv_heads=8, dim=128, page=32, window=0, mix=5),
        # The accepted tokens of one sequence.
        dict(name="keep_one", kind="keep", requests=1, context=531, nodes=7, kv_heads=8, dim=128,
             page=16, mix=6),
        # Those of many sequences with large trees.
        dict(name="keep_many", kind="keep", requests=128, context=1024, nodes=64, kv_heads=8,
             dim=128, page=64, mix=7),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "gated", "gated", "gated", "gated", "tree", "attend",
                       "attend", "attend", "attend", "keep"))
    elem = rng.choice(("f32", "f16", "bf16"))
    out = rng.choice(("elem", "q8_0"))
    mix = rng.randrange(1 << 20)
    if kind == "norm":
        dim = _log_uniform(rng, 64, 16384)
        dim = dim // 32 * 32 if out == "q8_0" or rng.random() < 0.7 else dim
        tokens = _log_uniform(rng, 1, 8192)
        return dict(kind=kind, elem=elem, tokens=min(tokens, MOST_NORM // dim), dim=dim, out=out)
    if kind == "gated":
        dim = _log_uniform(rng, 8, 512) * 32
        wide = _log_uniform(rng, 256, 16384)
        wide = wide // 32 * 32 if out == "q8_0" or rng.random() < 0.7 else wide
        wide = min(wide, MOST_WEIGHTS // (2 * dim) // 32 * 32)
        tokens = rng.choice((1, 1, 2, 3, _log_uniform(rng, 4, 64), _log_uniform(rng, 4, 64),
                             _log_uniform(rng, 65, 2048), _log_uniform(rng, 65, 2048)))
        return dict(kind=kind, elem=elem, act=rng.choice(("silu", "silu", "gelu_tanh", "gelu",
                                                          "relu")),
                    tokens=min(tokens, MOST_PRODUCTS // (2 * dim * wide)), dim=dim, wide=wide,
                    out=out)
    requests, nodes = _log_uniform(rng, 1, 256), _log_uniform(rng, 1, 128)
    if kind == "tree":
        return dict(kind=kind, requests=requests, nodes=nodes,
                    context=_log_uniform(rng, 1, 65536), mix=mix)
    page = rng.choice((16, 16, 32, 48, 64, 128))
    heads, kv_heads = rng.choice(((32, 8), (32, 32), (8, 1), (28, 4), (40, 8), (14, 2), (64, 8)))
    dim = rng.choice((64, 128, 128, 128, 192, 256))
    case = dict(kind=kind, elem=elem, requests=min(requests, 128),
                context=_log_uniform(rng, 16, 65536), nodes=nodes, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, window=0, mix=mix)
    if kind == "keep":
        case["context"] = min(case["context"], 4096)
        for name in ("elem", "heads", "window"):
            del case[name]
    elif rng.random() < 0.25:
        case["window"] = _log_uniform(rng, 16, 4096)
    heads = case.get("heads", kv_heads)
    while (case["requests"] * (case["context"] + case["nodes"]) * kv_heads * dim > MOST_CACHED * 1024
           or case["requests"] * (case["context"] + case["nodes"]) * heads * case["nodes"]
           > MOST_SCORES):
        if case["requests"] > 1 and (case["context"] < 2048 or rng.random() < 0.5):
            case["requests"] = max(1, case["requests"] * 3 // 4)
        elif case["context"] > 64:
            case["context"] = case["context"] * 3 // 4
        else:
            case["nodes"] = max(1, case["nodes"] * 3 // 4)
    return case


def _lengths(case):
    """[(length, nodes)] of the requests: tokens with the drafted ones, and the drafted ones.  The
    first request has the most of both; of many, one has no drafted token."""
    rng = random.Random(case["mix"])
    got = [(case["context"] + case["nodes"], case["nodes"])]
    for r in range(1, case["requests"]):
        nodes = 0 if r == 5 else rng.randint(max(1, case["nodes"] // 2), case["nodes"])
        got.append((rng.randint(max(1, case["context"] // 8), case["context"]) + nodes, nodes))
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


def _channels(gen, *shape):
    """The spread of a projection's channels: a few of them ten times the others."""
    spread = 0.5 + torch.rand(*shape, generator=gen, device=DEV)
    loud = torch.rand(*shape, generator=gen, device=DEV) < 0.03
    return torch.where(loud, spread * 10.0, spread)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _quantize_q4(x):
    """float32 [..., 32] -> Q4_0: (fp16 scales [...], uint8 quants [..., 32]).  The scale is the
    element of largest magnitude (the first of several) over -8."""
    mag = x.abs()
    place = torch.arange(32, device=x.device)
    first = torch.where(mag == mag.amax(-1, keepdim=True), place, 32).amin(-1, keepdim=True)
    d = x.gather(-1, first.clamp(max=31)) / -8.0
    inv = torch.where(d == 0, torch.zeros_like(d), torch.ones_like(d) / d)
    q = (x * inv + 8.5).floor().clamp(0, 15).to(torch.uint8)
    return d[..., 0].half(), q


def _quantize_q8(x):
    """float32 [..., 32] -> Q8_0: (fp16 scales [...], int8 quants [..., 32]): the largest magnitude
    over 127, quants to the nearest, halves to the even one.  The divisions are of tensors: by a
    number they may come as a product with its reciprocal."""
    top = x.abs().amax(-1, keepdim=True)
    d = top / torch.full_like(top, 127.0)
    inv = torch.where(d == 0, torch.zeros_like(d), torch.ones_like(d) / d)
    return d[..., 0].half(), (x * inv).round().to(torch.int8)


def _q4_rows(x):
    """float32 [rows, dim] -> Q4_0 rows, uint8 [rows, dim / 32 * 18]."""
    d, q = _quantize_q4(x.view(x.shape[0], -1, 32))
    packed = q[..., :16] | (q[..., 16:] << 4)
    return torch.cat((d[..., None].view(torch.uint8), packed), dim=-1).flatten(1).contiguous()


def _q8_rows(x):
    """float32 [rows, dim] -> Q8_0 rows, uint8 [rows, dim / 32 * 34]."""
    d, q = _quantize_q8(x.view(x.shape[0], -1, 32))
    return torch.cat((d[..., None].view(torch.uint8), q.view(torch.uint8)),
                     dim=-1).flatten(1).contiguous()


def _q4_values(rows, wide):
    """Q4_0 rows -> values [rows, dim] in the type `wide`."""
    blocks = rows.view(rows.shape[0], -1, 18)
    d = blocks[..., :2].contiguous().view(torch.float16).to(wide)
    q = torch.cat((blocks[..., 2:] & 15, blocks[..., 2:] >> 4), dim=-1).to(wide) - 8.0
    return (q * d).flatten(1)


def _q8_values(rows, wide):
    """Q8_0 rows -> values [rows, dim] in the type `wide`."""
    blocks = rows.view(rows.shape[0], -1, 34)
    d = blocks[..., :2].contiguous().view(torch.float16).to(wide)
    return (blocks[..., 2:].contiguous().view(torch.int8).to(wide) * d).flatten(1)


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


def _parents(case, seed):
    """[[parent of node j]] of the requests: chains that branch, several roots (-1) among them."""
    rng = random.Random(seed * 31 + case["mix"])
    got = []
    for _, nodes in _lengths(case):
        tree = []
        for j in range(nodes):
            tree.append(j - 1 if rng.random() < 0.5 else rng.randint(-1, j - 1))
        got.append(tree)
    return got


def _masks(parents, words):
    """[nodes of all requests][words] of 64 bits: of a node and its ancestors."""
    got = []
    for tree in parents:
        seen = []
        for j, p in enumerate(tree):
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        for bits in seen:
            row = [bits >> 64 * w & (1 << 64) - 1 for w in range(words)]
            got.append([w - (1 << 64) if w >> 63 else w for w in row])
    return got


def _requests(case, seed):
    """What a program that drafts has in hand: where its requests' tokens begin, their lengths, the
    pages of all of them, the tree's parents."""
    rows, page = _lengths(case), case.get("page", 16)
    first = [0]
    for _, nodes in rows:
        first.append(first[-1] + nodes)
    state = dict(first=_ints(first), length=_ints([length for length, _ in rows]),
                 tokens=first[-1], words=(case["nodes"] + 63) // 64,
                 parents=_ints([p for tree in _parents(case, seed) for p in tree]))
    held = [-(-length // page) for length, _ in rows]
    width, pages = max(held), sum(held) + 3
    shuffled = torch.randperm(pages, generator=_generator(seed), device=DEV).to(torch.int32)
    at = torch.arange(width, device=DEV)
    start = torch.cumsum(_ints([0] + held[:-1]).long(), 0)
    have = at[None] < _ints(held)[:, None]
    state["block_table"] = torch.where(
        have, shuffled[(start[:, None] + at).clamp(max=pages - 1)],
        torch.full((), -1, dtype=torch.int32, device=DEV)).contiguous()
    state.update(pages=pages, width=width)
    return state


def _cached(case, gen, length):
    """A request's quantized keys and values, [length, kv_heads, nb(, 32)]."""
    kv, nb = case["kv_heads"], case["dim"] // 32
    spread = _channels(gen, kv, case["dim"])
    k = _quantize_q4((_normal(gen, length, kv, case["dim"]) * spread).view(length, kv, nb, 32))
    v = _quantize_q4(_normal(gen, length, kv, case["dim"]).view(length, kv, nb, 32))
    return k, v


def _queries(case, seed, tokens):
    """Rows whose scores spread over a few units, as a trained head's do."""
    gen = _generator(seed * 7919 + 1)
    return (_normal(gen, tokens, case["heads"], case["dim"]) * 0.5).to(ELEM[case["elem"]])


def _paths(case, seed):
    """[[nodes of an accepted path, downwards]] of the requests: to a node that its draws choose."""
    rng = random.Random(seed * 37 + case["mix"])
    got = []
    for tree in _parents(case, seed):
        path, j = [], rng.randint(0, len(tree) - 1) if tree else -1
        while j >= 0:
            path.insert(0, j)
            j = tree[j]
        got.append(path)
    return got


def prepare(case, seed):
    kind = case["kind"]
    gen = _generator(seed)
    if kind == "norm":
        shape, elem = (case["tokens"], case["dim"]), ELEM[case["elem"]]
        spread = _channels(gen, case["dim"])
        return dict(case, x=(_normal(gen, *shape) * 0.3).to(elem),
                    residual=(_normal(gen, *shape) * spread).to(elem),
                    weight=1.0 + 0.2 * _normal(gen, case["dim"]))
    if kind == "gated":
        wide, dim = case["wide"], case["dim"]
        return dict(case, gate=_q4_rows(_normal(gen, wide, dim) * 0.02),
                    up=_q4_rows(_normal(gen, wide, dim) * 0.02),
                    rows=_q8_rows(_normal(gen, case["tokens"], dim) * _channels(gen, dim)))
    state = dict(case, **_requests(case, seed))
    if kind == "tree":
        return state
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    # what no token was stored in yet is 0xff
    state["cache"] = torch.full((state["pages"] * kv * page * dim * 9 // 8,), 255,
                                dtype=torch.uint8, device=DEV)
    gen = _generator(seed * 7919)
    for r, (length, _) in enumerate(_lengths(case)):
        at = torch.arange(length, device=DEV)
        slots = state["block_table"][r].long()[at // page] * page + at % page
        _place(state["cache"], page, kv, dim, slots, *_cached(case, gen, length))
    if kind == "attend":
        state["q"] = _queries(case, seed, state["tokens"])
        state["masks"] = torch.tensor(_masks(_parents(case, seed), state["words"]),
                                      dtype=torch.int64, device=DEV).view(-1, state["words"])
        return state
    paths = _paths(case, seed)
    state["count"] = _ints([len(p) for p in paths])
    state["path"] = _ints([p + [0] * (case["nodes"] - len(p)) for p in paths])
    # the drafted tokens' places, whose rows are read back: those kept, and the others as they were
    added = (state["first"][1:] - state["first"][:-1]).long()
    k = torch.arange(case["nodes"], device=DEV)
    at = (state["length"].long() - added)[:, None] + k
    slots = state["block_table"].long().gather(1, (at // page).clamp(max=state["width"] - 1))
    state["slots"] = (slots * page + at % page)[k < added[:, None]].contiguous()
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _norm(s):
    """(sum in the element type, norm in float32).  The mean of the squares in 64 bits, so that its
    root, rounded once, is the same in any order."""
    h = s["x"].float() + s["residual"].float()
    inverse = (1.0 / (h.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
    return h.to(s["x"].dtype), h * inverse * s["weight"]


def _activation(g, act):
    if act == "relu":
        return g.clamp(min=0.0)
    if act == "gelu":
        return 0.5 * g * torch.erfc(g * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return g / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))
    return g / (1.0 + torch.exp(-g))


def _gated(s):
    x = _q8_values(s["rows"], torch.float32)
    gate = torch.matmul(x, _q4_values(s["gate"], torch.float32).t())
    up = torch.matmul(x, _q4_values(s["up"], torch.float32).t())
    return _activation(gate, s["act"]) * up


def _blocks(x):
    """The values that Q8_0 blocks of x stand for, float32."""
    d, q = _quantize_q8(x.view(x.shape[0], -1, 32))
    return (q.float() * d.float()[..., None]).flatten(1)


def _tree(s):
    """masks int64 [tokens, words] and positions int32 [tokens].  A node's depth is that of its
    parent and one: rounds in which every node takes its parent's ancestors, the reach of a node
    twice as far in each."""
    first, tokens, words = s["first"].long(), s["tokens"], s["words"]
    i = torch.arange(tokens, device=DEV)
    r = torch.searchsorted(first[1:], i, right=True)
    j = i - first[r]
    bit = torch.where((j[:, None] // 64) == torch.arange(words, device=DEV),
                      torch.ones_like(j)[:, None] << (j[:, None] % 64), 0)
    # row `tokens` is the ancestor of a root: it sees nothing and is its own ancestor
    up = torch.where(s["parents"] < 0, tokens, first[r] + s["parents"].long())
    up = torch.cat((up, torch.full_like(up[:1], tokens)))
    masks = torch.cat((bit, torch.zeros_like(bit[:1])))
    depth = torch.cat(((s["parents"] >= 0).long(), torch.zeros_like(j[:1])))
    for _ in range(max(1, s["nodes"].bit_length())):
        masks, depth, up = masks | masks[up], depth + depth[up], up[up]
    before = s["length"].long() - (first[1:] - first[:-1])
    return dict(masks=masks[:-1], positions=(before[r] + depth[:-1]).int())


def _bits(masks):
    """int64 [n, words] -> truth values [n, words * 64]."""
    return ((masks[..., None] >> torch.arange(64, device=DEV)) & 1).bool().flatten(1)


def _attend(s):
    """float32 [tokens, heads, dim]: softmax(q k' / sqrt(dim)) v over what each drafted token sees:
    its request's cached tokens, of them those that the window leaves, and its ancestors."""
    heads, kv, dim, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    n, most, q = s["block_table"].shape[0], s["nodes"], s["q"]
    first, length = s["first"].long(), s["length"].long()
    slots = (s["block_table"].clamp(min=0).long()[..., None] * page
             + torch.arange(page, device=DEV)).reshape(-1)
    k, v = _read(s["cache"], page, kv, dim, slots)
    k, v = (x.view(n, -1, kv, dim).transpose(1, 2) for x in (k, v))
    t = torch.arange(k.shape[2], device=DEV)
    v = torch.where((t < length[:, None])[:, None, :, None], v, torch.zeros_like(v))
    added = first[1:] - first[:-1]
    i = torch.arange(most, device=DEV)
    token = (first[:-1, None] + i).clamp(max=q.shape[0] - 1)
    rows = q.float()[token].view(n, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(rows.reshape(n, kv, -1, dim) * dim ** -0.5, k.transpose(2, 3))
    before = (length - added)[:, None, None]
    tree = _bits(s["masks"])[token]                              # [n, most, words * 64]
    depth = tree.long().cumsum(-1) - 1                           # of an ancestor
    place = (t[None, None] - before).clamp(0, tree.shape[-1] - 1).expand(n, most, -1)
    seen = torch.where(t < before, True, tree.gather(2, place)) & (t < length[:, None, None])
    if s["window"]:
        position = torch.where(t < before, t.expand(n, most, -1), before + depth.gather(2, place))
        seen = seen & (position > before + depth[..., -1:] - s["window"])
    scores = scores.view(n, kv, -1, most, t.shape[0])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, kv, -1, t.shape[0]), v).view(n, kv, -1, most, dim)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 3, 1, 2, 4).reshape(n, most, heads, dim)[i < added[:, None]]


def _keep(s):
    """The accepted nodes' rows to the places after the cached ones, all read before one is written."""
    page, table = s["page"], s["block_table"].long()
    before = (s["length"].long() - (s["first"][1:] - s["first"][:-1]).long())[:, None]
    k = torch.arange(s["nodes"], device=DEV)
    kept = k < s["count"][:, None]

    def slots(at):
        at = torch.where(kept, at, torch.zeros_like(at))
        return (table.gather(1, at // page) * page + at % page)[kept]

    source, to = slots(before + s["path"]), slots(before + k)
    page_at, off, group, lane = source // page, source % page, source % page // 4, source % 4
    kq, ks, vq, vs = _views(s["cache"], page, s["kv_heads"], s["dim"])
    took = (kq[page_at, :, off], ks[page_at, :, group, :, lane], vq[page_at, :, group, :, :, lane],
            vs[page_at, :, group, :, lane])
    page_at, off, group, lane = to // page, to % page, to % page // 4, to % 4
    kq[page_at, :, off] = took[0]
    ks[page_at, :, group, :, lane] = took[1]
    vq[page_at, :, group, :, :, lane] = took[2]
    vs[page_at, :, group, :, lane] = took[3]


def _plain(s):
    kind = s["kind"]
    if kind == "norm":
        total, y = _norm(s)
        return dict(sum=total, y=_blocks(y) if s["out"] == "q8_0" else y.to(total.dtype))
    if kind == "gated":
        y = _gated(s)
        return _blocks(y).half() if s["out"] == "q8_0" else y.to(ELEM[s["elem"]])
    if kind == "tree":
        return _tree(s)
    if kind == "attend":
        return _attend(s).to(ELEM[s["elem"]])
    _keep(s)
    k, v = _read(s["cache"], s["page"], s["kv_heads"], s["dim"], s["slots"])
    return dict(k=k, v=v)


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


def _buffers(s, rows, dim, dtype):
    """Rows of an element type or of Q8_0 blocks, and (for those) their values."""
    if s["out"] == "elem":
        return s.setdefault("made", (torch.empty(rows, dim, dtype=dtype, device=DEV), None, None))
    return s.setdefault("made", (None, torch.empty(rows, dim // 32 * 34, dtype=torch.uint8,
                                                   device=DEV),
                                 torch.empty(rows, dim, dtype=torch.float32, device=DEV)))


def _framework(s):
    hip, kind = _binding(), s["kind"]
    if kind == "norm":
        x, residual, tokens, dim = s["x"], s["residual"], s["tokens"], s["dim"]
        total = s.setdefault("sum", torch.empty_like(x))
        y, q8, values = _buffers(s, tokens, dim, x.dtype)
        hip.add_rms_norm(s["elem"], x, dim, residual, dim, total, dim, s["weight"], EPS, y, dim,
                         q8, dim // 32 * 34, tokens, dim)
        if q8 is None:
            return dict(sum=total, y=y)
        hip.dequantize_row_q8_0(q8, values, tokens * dim)
        return dict(sum=total, y=values)
    if kind == "gated":
        tokens, dim, wide = s["tokens"], s["dim"], s["wide"]
        out, q8, values = _buffers(s, tokens, wide, ELEM[s["elem"]])
        hip.gated_q4_0_q8_0(s["elem"], s["act"], dim, out, wide, q8, wide // 32 * 34, s["gate"],
                            s["up"], dim // 32 * 18, s["rows"], dim // 32 * 34, wide, tokens)
        if q8 is None:
            return out
        hip.dequantize_row_q8_0(q8, values, tokens * wide)
        return values.half()
    n, tokens, words = s["first"].shape[0] - 1, s["tokens"], s["words"]
    if kind == "tree":
        masks, positions = s.setdefault("made", (
            torch.empty(tokens, words, dtype=torch.int64, device=DEV),
            torch.empty(tokens, dtype=torch.int32, device=DEV)))
        hip.tree_tables(s["parents"], s["first"], s["length"], n, masks, words, positions, tokens)
        return dict(masks=masks, positions=positions)
    kv, dim, page = s["kv_heads"], s["dim"], s["page"]
    if kind == "attend":
        q, heads, most = s["q"], s["heads"], s["context"] + s["nodes"]
        if "out" not in s:
            need = hip.attn_tree_q4_0_workspace_bytes(s["elem"], n, tokens, s["nodes"], most,
                                                      heads, kv, dim)
            s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
            s["out"] = torch.empty_like(q)
        out = s["out"]
        hip.attn_tree_q4_0(s["elem"], q, q.stride(0), q.stride(1), s["cache"], s["pages"], page,
                           s["block_table"], s["width"], s["first"], s["length"], s["masks"],
                           words, n, tokens, s["nodes"], most, heads, kv, dim, dim ** -0.5,
                           s["window"], out, out.stride(0), out.stride(1), s["workspace"],
                           s["workspace"].numel())
        return out
    hip.kv_keep_q4_0(s["cache"], s["pages"], page, s["block_table"], s["width"], s["first"],
                     s["length"], s["path"], s["nodes"], s["count"], n, s["nodes"], kv, dim)
    kept = s["slots"].shape[0]
    k, v = s.setdefault("read", (torch.empty(kept, kv, dim, device=DEV),
                                 torch.empty(kept, kv, dim, device=DEV)))
    hip.kv_load_q4_0("f32", s["cache"], s["pages"], page, s["slots"], k, k.stride(0), k.stride(1),
                     v, v.stride(0), v.stride(1), kept, kv, dim)
    return dict(k=k, v=v)


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# The least work, and the results in float64
# ---------------------------------------------------------------------------

def work(case):
    kind, size = case["kind"], {"f32": 4}.get(case.get("elem"), 2)
    if kind == "norm":
        n, q8 = case["tokens"] * case["dim"], case["out"] == "q8_0"
        # read back, the blocks' values are four bytes each
        return {"bytes": 3 * n * size + 4 * case["dim"] + (2 * n * 34 // 32 + 4 * n if q8
                                                           else n * size), "flops": 5 * n}
    if kind == "gated":
        n, weights = case["tokens"] * case["wide"], 2 * case["wide"] * case["dim"]
        out = 2 * n * 34 // 32 + 10 * n if case["out"] == "q8_0" else n * size
        return {"bytes": weights * 9 // 16 + case["tokens"] * case["dim"] * 34 // 32 + out,
                "flops": 2 * weights * case["tokens"]}
    rows = _lengths(case)
    nodes, words = sum(n for _, n in rows), (case["nodes"] + 63) // 64
    if kind == "tree":
        return {"bytes": len(rows) * 8 + nodes * (8 + 8 * words), "flops": nodes}
    row = case["kv_heads"] * case["dim"] * 9 // 8
    if kind == "keep":
        # of each tree one node at least is kept; all of its places are read back
        kept = sum(1 for _, n in rows if n)
        return {"bytes": len(rows) * 12 + kept * (4 + 2 * row)
                + nodes * (8 + row + 8 * case["kv_heads"] * case["dim"]), "flops": kept}
    heads, dim = case["heads"], case["dim"]
    cached = pairs = 0
    for length, n in rows:
        begin = max(0, length - n - case["window"] + 1) if case["window"] else 0
        if n:
            cached += length - begin
            pairs += n * (length - n - begin) + n
    return {"bytes": cached * row + 2 * nodes * heads * dim * size + nodes * 8 * words
            + len(rows) * 8, "flops": 4 * pairs * heads * dim}


def _exact_blocks(y):
    """What Q8_0 blocks of float64 rows stand for, float64: scales are the blocks' own, in fp16."""
    blocks = y.view(y.shape[0], -1, 32)
    top = blocks.abs().amax(-1, keepdim=True)
    quants = torch.where(top > 0, torch.round(blocks * 127.0 / top.clamp(min=1e-300)), 0.0)
    return (quants * (top / 127.0).half().double()).flatten(1)


def _exact_activation(g, act):
    if act == "relu":
        return torch.relu(g)
    if act == "gelu":
        return g * 0.5 * (1.0 + torch.erf(g / math.sqrt(2.0)))
    if act == "gelu_tanh":
        return g * 0.5 * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
    return g * torch.sigmoid(g)


def _exact_attention(case, q, k, v, length, tree):
    """One request's rows in float64: q [nodes, heads, dim], k and v [length, kv_heads, dim], and
    the parents of its nodes."""
    nodes, before = len(tree), length - len(tree)
    hidden = torch.zeros(nodes, length, dtype=torch.bool)
    hidden[:, before:] = True
    for j in range(nodes):
        path, p = [], j
        while p >= 0:
            path.append(p)
            p = tree[p]
        depth = len(path) - 1
        for up, p in enumerate(path):  # `up` above j
            hidden[j, before + p] = bool(case["window"]) and up >= case["window"]
        if case["window"]:
            hidden[j, :max(0, min(before, before + depth - case["window"] + 1))] = True
    hidden = hidden.to(DEV)
    out = torch.empty(nodes, case["heads"], case["dim"], dtype=torch.float64, device=DEV)
    share = case["heads"] // case["kv_heads"]
    for h in range(case["heads"]):
        z = (q[:, h] @ k[:, h // share].t()) / math.sqrt(case["dim"])
        out[:, h] = torch.softmax(z.masked_fill(hidden, -math.inf), dim=1) @ v[:, h // share]
    return out


def _wide(part):
    return ((part[1].double() - 8.0) * part[0].double()[..., None]).flatten(-2)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("tree", "keep"):  # whole numbers, and bytes that are moved, have no other
        return None
    if kind == "norm":
        s = prepare(case, seed)
        total = s["x"].double() + s["residual"].double()
        if case["out"] == "q8_0":  # the blocks are those of the norm in 32 bits
            return dict(sum=total, y=None)
        y = total / (total.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["weight"].double()
        return dict(sum=total, y=y)
    if kind == "gated":
        s = prepare(case, seed)
        x = _q8_values(s["rows"], torch.float64).t().contiguous()
        gate, up = ((_q4_values(s[m], torch.float64) @ x).t() for m in ("gate", "up"))
        y = _exact_activation(gate, case["act"]) * up
        return _exact_blocks(y.contiguous()) if case["out"] == "q8_0" else y
    rows, trees = _lengths(case), _parents(case, seed)
    gen = _generator(seed * 7919)
    q = _queries(case, seed, sum(n for _, n in rows)).double()
    got, at = [], 0
    for (length, nodes), tree in zip(rows, trees):
        k, v = (_wide(part) for part in _cached(case, gen, length))
        if nodes:
            got.append(_exact_attention(case, q[at:at + nodes], k, v, length, tree))
        at += nodes
    return torch.cat(got)
