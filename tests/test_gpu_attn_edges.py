"""attn_q4_0 where a row sees little or what it sees is uneven.  Oracle and, where not said otherwise,
tolerances: those of test_gpu_kv_cache.Setup (float64)."""
import numpy as np
import pytest

import kv_plain
from test_gpu_kv_cache import ELEMS, Setup, wide

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------- missing pages ---

def attend_there(q, keys, vals, position0, scale, causal, window, there):
    """kv_plain.attend with the tokens alone that `there` holds, for all rows of a head at once."""
    added, heads, dim = q.shape
    length, kv, _ = keys.shape
    at, t = position0 + np.arange(added)[:, None], np.arange(length)[None]
    seen = np.broadcast_to(there, (added, length)).copy()
    if causal:
        seen &= t <= at
    if window:
        seen &= t > at - window
    out = np.zeros((added, heads, dim))
    some = seen.any(1)
    for h in range(heads):
        z = scale * (q[:, h].astype(np.float64) @ keys[:, h * kv // heads].T)
        z = np.where(seen, z, -np.inf)[some]
        w = np.exp(z - z.max(1, keepdims=True))
        out[some, h] = w @ vals[:, h * kv // heads] / w.sum(1, keepdims=True)
    return out, some


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("lengths,added,heads,kv,page,holes", [
    # whole tiles; the last page in part, and a request of nothing else
    ([150, 70, 33], [150, 70, 33], 12, 2, 16, [(0, 3, 4, 9), range(5), ()]),
    # pages of three halves of a step
    ([400], [130], 8, 1, 48, [(0, 2, 5, 8)]),
    # parts of a context
    ([4500], [20], 2, 1, 16, [(0, 7, *range(100, 121), 130, 281)]),
    # beside requests of few rows
    ([2000, 1500, 900, 40], [1, 300, 2, 40], 8, 2, 32, [(1, 2), (0, 30, 46), (5,), (1,)]),
])
def test_prompts_with_missing_pages(hip, dev, elem, dim, lengths, added, heads, kv, page, holes):
    """Tokens of a page outside the cache are not there, in prompts as in single tokens."""
    s = Setup(dev, elem, lengths, added, heads, kv, dim, page, seed=21)
    table = s.table.copy()
    for r, pages in enumerate(holes):
        for i, page_at in enumerate(pages):
            table[r, page_at] = -1 if i % 2 == 0 else s.pages
    for causal, window in ((True, 0), (False, 0), (True, 90), (True, 9)):
        out = wide(s.run(hip, table=table, causal=causal, window=window))
        want, some = zip(*(
            attend_there(s.q[s.first[r]:s.first[r + 1]], s.k[r], s.v[r], lengths[r] - added[r],
                         np.float64(np.float32(dim ** -0.5)), causal, window,
                         ~np.isin(np.arange(lengths[r]) // page, list(holes[r])))
            for r in range(len(lengths))))
        want, some = np.concatenate(want), np.concatenate(some)
        off = np.abs(out - want)
        assert (off <= s.tolerance(want)).all(), (causal, window, off.max())
        assert (out[~some] == 0.0).all()


# ------------------------------------------------- rows that are not finite ---

@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length,added", [(90, 90), (20, 30), (9, 4)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_bad_rows(hip, dev, elem, dim, length, added, bad):
    """A row that holds an infinity or a NaN is NaN whatever it sees, one token or many, and zero
    where it sees none; the other rows keep their bits."""
    s = Setup(dev, elem, [length], [added], 4, 1, dim, 16, seed=22)
    clean = s.q.copy()
    place = np.zeros((added, 4), bool)
    for i in range(added):
        for h in (1, 3) if i % 3 else (0, 1, 2):
            s.q[i, h, (11 * i + 17 * h) % dim] = bad
            place[i, h] = True
    sees = length - added + np.arange(added) >= 0
    for window in (0, 1):
        got = wide(s.run(hip, window=window))
        kept, s.q = s.q, clean
        fine = wide(s.run(hip, window=window))
        s.q = kept
        assert np.isnan(got[place & sees[:, None]]).all()
        assert (got[~sees] == 0.0).all()
        assert np.array_equal(got[~place], fine[~place])


# -------------------------------------------------------- query magnitudes ---

@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("power", [-122, -105, 105, 122])
@pytest.mark.parametrize("added", [3, 60])
def test_queries_of_any_power(hip, dev, elem, power, added):
    """Rows near either end of the type's range, with the scale that brings their scores back."""
    s = Setup(dev, elem, [200], [added], 4, 1, 64, 16, seed=23, spread=2.0 ** power)
    s.check(hip, scale=0.1 * 2.0 ** -power)


# ------------------------------------------------------- loud beside quiet ---

class Shared(Setup):
    """Requests that share one run of cached tokens, a new token and one query head each: so many
    that a work-group takes a whole context and one wave a quarter of it."""

    def __init__(self, dev, elem, k, v, q, requests=512, page=64):
        length, kv, dim = k.shape
        super().__init__(dev, elem, [length], [1], 1, kv, dim, page)
        kq, vq = kv_plain.quantize(k.astype(np.float32)), kv_plain.quantize(v.astype(np.float32))
        self._put(self.cache, self.slots, kq, vq)
        self.one = kv_plain.values(*kq)[:, 0], kv_plain.values(*vq)[:, 0]
        self.lengths, self.added = (np.full(requests, n, np.int32) for n in (length, 1))
        self.table = np.repeat(self.table, requests, 0)
        self.first, self.tokens = np.arange(requests + 1, dtype=np.int32), requests
        self.q = kv_plain.round_to(np.broadcast_to(q, (requests, 1, dim)).copy(), elem)

    def weights(self):
        """The softmax over the tokens, float64."""
        z = self.one[0] @ self.q[0, 0].astype(np.float64) * np.float64(np.float32(self.dim ** -0.5))
        w = np.exp(z - z.max())
        return w / w.sum()


def sink(dev, elem, dim, at, value_of, tail):
    """2560 tokens, all of a weight of 2^-19 but the one at `at`, which has nearly all of it.
    tail: magnitudes of the values of elements 32 .. 63; value_of: loud ones, {token: value}, of
    element 0."""
    rng = np.random.default_rng(24)
    k = np.zeros((2560, 1, dim))
    k[at, 0, 0] = 4.0
    v = np.zeros((2560, 1, dim))
    v[:, 0, 32:64] = tail * rng.uniform(0.5, 1.0, (2560, 32))
    v[at, 0, 32:64] = 0.0
    for token, value in value_of.items():
        v[token, 0, 0] = value
    q = np.zeros(dim)
    q[0] = 19.0 * np.log(2.0) * dim ** 0.5 / 4.0
    return Shared(dev, elem, k, v, q)


def check_tail(hip, s, top_scale):
    """Elements 32 .. 63.  A weight is off by twice 2^-21 |z| (z up to 13.2 here) and 2^-20 of it; a
    weight times a scale is rounded to 11 bits for 16-bit rows, to 22 for f32, and at 2^-25 of what
    brings weight and largest scale to 2^15 at most and over 2^10: to 2^-35 of that scale.  Eight
    times that a token at most."""
    out = wide(s.run(hip))[:, 0, 32:64]
    w, v = s.weights(), s.one[1][:, 32:64]
    want, mass = w @ v, w @ np.abs(v)
    tol = mass * (2.0 ** -22 if s.elem == "f32" else 2.0 ** -11)
    tol += mass * 2 * (2.0 ** -21 * 13.2 + 2.0 ** -20) + 8 * len(w) * top_scale * 2.0 ** -35
    tol += np.abs(want) * {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[s.elem]
    off = np.abs(out - want)
    assert (off <= tol).all(), (off.max(), tol.min(), want.mean())


@pytest.mark.parametrize("elem", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("at", [0, 1300])
def test_tail_of_small_values(hip, dev, elem, dim, at):
    """Values of 2^-14 and less under weights that are small together and not alone."""
    check_tail(hip, sink(dev, elem, dim, at, {}, 2.0 ** -14), 2.0 ** -12)  # scales below 2^-11 alike


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("at,loud", [
    (0, {0: 32.0}), (1300, {1300: 32.0}), (1300, {100: 32.0, 1300: -512.0}), (40, {41: 20.0}),
])
def test_tail_beside_loud_values(hip, dev, elem, dim, at, loud):
    """Values of 1 in one block where another has some of 20 to 512."""
    top = max(abs(x) for x in loud.values()) / 8
    check_tail(hip, sink(dev, elem, dim, at, loud, 1.0), top)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("at,token", [(0, 0), (0, 700), (1300, 1301)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_tail_beside_a_scale_that_is_not_finite(hip, dev, elem, dim, at, token, bad):
    """Values of 1 in one block where another has a scale that is not finite: they keep their weights,
    as beside scales below 2."""
    s = sink(dev, elem, dim, at, {}, 1.0)
    lay, (page, t) = s.cache, divmod(int(s.slots[token]), s.page)
    o = 2 * lay.quants + lay.scales + (t // 4) * lay.nb * 8 + (t % 4) * 2
    lay.bytes[page, 0, o:o + 2] = np.array([bad], np.float16).view(np.uint8)
    check_tail(hip, s, 1.0)
    assert not np.isfinite(wide(s.run(hip))[:, 0, :32]).any()


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
def test_prompt_keys_beside_a_loud_one(hip, dev, elem, dim):
    """Small keys under a large scale of the scores, and after them one key of 2^6: the rows before
    it do not see it, and keep all bits of theirs."""
    s = Setup(dev, elem, [100], [100], 4, 1, dim, 16, seed=25)
    rng = np.random.default_rng(25)
    k = rng.standard_normal((100, 1, dim)) * 2.0 ** -12
    k[99] *= 2.0 ** 18
    kq, vq = kv_plain.quantize(k.astype(np.float32)), kv_plain.quantize(s.v[0].astype(np.float32))
    s._put(s.cache, s.slots, kq, vq)
    s.k, s.v = [kv_plain.values(*kq)], [kv_plain.values(*vq)]
    scale = 2.0 ** 9
    out, want = wide(s.run(hip, scale=scale))[:99], s.want(scale=scale)[:99]
    s.k = [s.k[0][:99]]  # those whose norm counts
    off = np.abs(out - want)
    assert (off <= s.tolerance(want, scale)).all(), off.max()


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("loud", [{3: 64.0}, {70: 64.0}, {99: 64.0}, {3: 64.0, 70: 40000.0},
                                  {70: 40000.0}])
@pytest.mark.parametrize("length,added", [(100, 100), (1100, 20)])
def test_prompt_values_beside_loud_ones(hip, dev, elem, dim, loud, length, added):
    """Values of 2^-12 in block 1, in a prompt whose block 0 has single large ones; each block by
    its own values.  Past scales of 4096 a value ends at 2^-21."""
    s = Setup(dev, elem, [length], [added], 8, 1, dim, 16, seed=26)
    rng = np.random.default_rng(26)
    v = rng.standard_normal((length, 1, dim))
    v[:, :, 32:64] *= 2.0 ** -12
    for token, value in loud.items():
        v[token, 0, 5] = value
    kq, vq = kv_plain.quantize(s.k[0].astype(np.float32)), kv_plain.quantize(v.astype(np.float32))
    s._put(s.cache, s.slots, kq, vq)
    s.k, s.v = [kv_plain.values(*kq)], [kv_plain.values(*vq)]
    out, want = wide(s.run(hip)), s.want()
    whole = s.v[0]
    for b in range(dim // 32):
        block = slice(32 * b, 32 * b + 32)
        s.v = [whole[:, :, block]]
        tol = s.tolerance(want[..., block]) + (2.0 ** -25 if elem == "f16" else 0.0)
        tol += 2.0 ** -21 if max(loud.values()) > 32768 else 0.0
        off = np.abs(out - want)[..., block]
        assert (off <= tol).all(), (b, off.max())


# ------------------------------------------------------------- wide windows ---

@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("lengths,added", [([20, 50], [30, 3]), ([3, 1], [6, 1])])
def test_windows_wider_than_all_positions(hip, dev, elem, lengths, added):
    """They hide nothing, also from rows before the first position, which see all tokens where a row's
    own position is no bound."""
    s = Setup(dev, elem, lengths, added, 4, 2, 64, 16, seed=27)
    for causal in (False, True):
        whole = wide(s.run(hip, causal=causal))
        for window in (2 ** 30, 2 ** 31 - 20, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 32 + 1):
            assert np.array_equal(wide(s.run(hip, causal=causal, window=window)), whole), window
    s.check(hip, causal=False)


# ------------------------------------------------------- error of 16-bit rows ---

@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("length,added", [(700, 200), (1500, 90)])
def test_error_of_f16_prompts(hip, dev, dim, length, added):
    """The error against float64, as a 2-norm, is that of the roundings that are meant: values to f16,
    every other 16 tokens' weights to f16, the output to f16.  Their sum is formed here from the same
    inputs, with weights over the row's own maximum; the kernel's base differs, which shifts which
    weights round up and which down: 3 % for that, where rounding the others' too adds 7 %."""
    s = Setup(dev, "f16", [length], [added], 8, 2, dim, 16, seed=28, spread=0.5)
    out, want = wide(s.run(hip)), s.want()
    model = np.empty_like(want)
    at, t = length - added + np.arange(added)[:, None], np.arange(length)[None]
    half = np.float64(2.0 ** 10)
    values = (s.v[0] * half).astype(np.float16).astype(np.float64) / half
    for h in range(8):
        z = np.float64(np.float32(dim ** -0.5)) * (s.q[:, h].astype(np.float64) @ s.k[0][:, h // 4].T)
        z = np.where(t <= at, z, -np.inf)
        w = np.exp(z - z.max(1, keepdims=True)) * half
        w = np.where(t // 16 % 2 == 0, w.astype(np.float16).astype(np.float64), w)
        model[:, h] = w @ values[:, h // 4] / w.sum(1, keepdims=True)
    model = model.astype(np.float16).astype(np.float64)
    assert np.linalg.norm(out - want) <= 1.03 * np.linalg.norm(model - want)
