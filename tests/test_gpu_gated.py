"""gated_q4_0_q8_0 on the GPU against its formula in float64, and its Q8_0 blocks against the quantizer over
its own float32 outputs.

How far an output may be off, eps = 2^-24: a projection is a sum of nb terms, each rounded when it is scaled
(one step) and at most nb times while it is added, so off by (nb + 1) eps of the sum of its terms'
magnitudes.  The activations' derivatives are at most 1.13; their own evaluation is off by 8 eps of the value
for a quotient of a sum with one exponential (2 steps of its own, 1 each of the sum and the quotient, the
rest for the product with u and the argument's rounding), by 3 eps |x| more where the exponential's argument
x is itself rounded (three steps of the tanh form's, one of silu's: none), and for the complement of the
error function, of relative condition 2 z^2 = g^2, by (32 + 2 g^2) eps.  The output's own rounding is half
a step of its type."""
import numpy as np
import pytest
import torch

import synth
from gpu_util import from_dev, to_dev
from test_gpu_kv_cache import ELEMS, TORCH, wide

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu_tanh", "gelu", "relu"]
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def q4_blocks(rows):
    b = rows.reshape(rows.shape[0], -1, 18)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    return np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8.0, d


def q8_blocks(rows):
    b = rows.reshape(rows.shape[0], -1, 34)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    return np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64), d


def project(w, y):
    """(values, sums of the terms' magnitudes) [tokens][features] in float64."""
    (qw, dw), (qy, dy) = q4_blocks(w), q8_blocks(y)
    total = np.zeros((y.shape[0], w.shape[0]))
    size = np.zeros_like(total)
    for b in range(qw.shape[1]):
        t = (qy[:, b] @ qw[:, b].T) * dy[:, b] * dw[:, b, 0]
        total += t
        size += np.abs(t)
    return total, size


def erfc(z):
    from scipy.special import erfc as f
    return f(z)


def activation(g, act):
    """(value, what its evaluation may be off by, in steps of 2^-24)."""
    if act == "relu":
        return np.maximum(g, 0.0), 0.0
    if act == "gelu":
        v = 0.5 * g * erfc(-g / np.sqrt(2.0))
        return v, (32 + 2 * g * g) * np.abs(v)
    x = g if act == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
    v = g * (np.exp(x) / (1 + np.exp(x)) if np.ndim(x) == 0 else np.where(
        x < 0, np.exp(np.minimum(x, 0)) / (1 + np.exp(np.minimum(x, 0))),
        1 / (1 + np.exp(-np.maximum(x, 0)))))
    return v, (8 + (0 if act == "silu" else 3 * np.abs(x))) * np.abs(v)


def want_of(gate, up, y, act, elem):
    nb, eps = y.shape[1] // 34, 2.0 ** -24
    (g, gs), (u, us) = project(gate, y), project(up, y)
    a, steps = activation(g, act)
    v = a * u
    off = np.abs(u) * (1.13 * (nb + 1) * eps * gs + steps * eps) + np.abs(a) * (nb + 1) * eps * us
    off += 1.13 * (nb + 1) ** 2 * eps ** 2 * gs * us + 2 * eps * np.abs(v)
    return v, off * 1.001 + HALF[elem] * np.abs(v) + LEAST[elem]


class Case:
    def __init__(self, n, wide_, tokens, seed=0, apart=(0, 0), layout="apart"):
        self.n, self.wide, self.tokens = n, wide_, tokens
        self.gate = synth.q4_0_matrix(wide_, n, 50 + seed, 1.5 * n ** -0.5)
        self.up = synth.q4_0_matrix(wide_, n, 51 + seed, 1.5 * n ** -0.5)
        self.y = synth.q8_0_matrix(tokens, n, 52 + seed, 1.0)
        self.apart, self.layout = apart, layout

    def run(self, hip, dev, elem, act, out=True, q8=True, stream=None):
        """(out, q8) on the host, checked to have left what lies between the rows."""
        xpad, ypad = self.apart
        bw, by = self.n // 32 * 18, self.n // 32 * 34
        if self.layout == "apart":
            bx = bw + xpad
            buf = np.full(2 * self.wide * bx, 0xEE, np.uint8)
            both = buf.reshape(2, self.wide, bx)
            both[0, :, :bw], both[1, :, :bw] = self.gate, self.up
            dw = to_dev(buf, dev)
            gate, up = dw, dw[self.wide * bx:]
        else:  # rows in turn
            bx = 2 * bw
            dw = to_dev(np.stack([self.gate, self.up], 1), dev).view(-1)
            gate, up = dw, dw[bw:]
        rows = np.full((self.tokens, by + ypad), 0xEE, np.uint8)
        rows[:, :by] = self.y
        dy = to_dev(rows, dev)
        nb, step = self.wide // 32, self.wide + 3 * (xpad // 2)
        row8 = nb * 34 + xpad
        to = torch.full((self.tokens * step + 8,), 7.0, dtype=TORCH[elem], device=dev)
        to8 = torch.full((self.tokens * row8 + 16,), 0xEE, dtype=torch.uint8, device=dev)
        hip.gated_q4_0_q8_0(elem, act, self.n, to if out else None, step, to8 if q8 else None, row8,
                            gate, up, bx, dy, by + ypad, self.wide, self.tokens, stream)
        got, got8 = wide(to), from_dev(to8)
        a = got[:self.tokens * step].reshape(self.tokens, step)
        b = got8[:self.tokens * row8].reshape(self.tokens, row8)
        assert (a[:, self.wide if out else 0:] == 7.0).all() and (got[self.tokens * step:] == 7.0).all()
        assert (b[:, nb * 34 if q8 else 0:] == 0xEE).all() and (got8[self.tokens * row8:] == 0xEE).all()
        return a[:, :self.wide], b[:, :nb * 34]

    def check(self, hip, dev, elem, act, q8=True):
        got, got8 = self.run(hip, dev, elem, act, q8=q8)
        want, tol = want_of(self.gate, self.up, self.y, act, elem)
        off = np.abs(got - want)
        assert np.isfinite(got).all()
        assert (off <= tol).all(), (off / tol).max()
        whole = self.wide // 32 * 32
        exact = got if elem == "f32" or not q8 else self.run(hip, dev, "f32", act)[0]
        if whole and q8:
            assert np.array_equal(got8.reshape(-1),
                                  synth.quantize_q8_0(np.ascontiguousarray(exact[:, :whole])))
        return got


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 31, 32, 33, 70])
@pytest.mark.parametrize("n,wide_", [(32, 32), (64, 33), (96, 31), (288, 100), (2080, 64)])
def test_sizes(hip, dev, elem, tokens, n, wide_):
    Case(n, wide_, tokens).check(hip, dev, elem, "silu")


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 33, 70])
@pytest.mark.parametrize("n,wide_", [(32, 15), (64, 33), (96, 48), (544, 2050), (288, 4100), (2080, 64)])
def test_elements_alone(hip, dev, elem, tokens, n, wide_):
    Case(n, wide_, tokens, seed=2).check(hip, dev, elem, "silu", q8=False)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("tokens,n,wide_", [
    (1, 4096, 1000), (4, 4128, 320), (9, 4096, 257), (129, 512, 130), (150, 1056, 129),
    (300, 256, 384), (513, 544, 200), (1000, 128, 65), (1, 32, 1), (200, 32, 1), (6, 14336, 40),
    (1, 14336, 40), (2, 20000, 33),
])
def test_larger_and_ragged(hip, dev, elem, tokens, n, wide_):
    Case(n, wide_, tokens, seed=3).check(hip, dev, elem, "silu")


# Many features and tokens, where tiles of 64 and of 128 features serve (tests/test_more_dispatch.py holds that),
# ragged both ways.
TILES = {"tiles of 64": (500, 4090), "tiles of 128": (630, 4590)}


@pytest.mark.parametrize("elem,n", [("f32", 32), ("f32", 96), ("f32", 1056), ("f16", 224), ("bf16", 416)])
@pytest.mark.parametrize("tiles", TILES)
def test_tiles(hip, dev, elem, n, tiles):
    tokens, wide_ = TILES[tiles]
    Case(n, wide_, tokens, seed=4).check(hip, dev, elem, "silu")


@pytest.mark.parametrize("apart,layout", [((2, 2), "apart"), ((14, 34), "apart"), ((0, 0), "in turn")])
@pytest.mark.parametrize("tiles", TILES)
def test_tiles_of_strided_rows(hip, dev, apart, layout, tiles):
    tokens, wide_ = TILES[tiles]
    Case(160, wide_, tokens, seed=6, apart=apart, layout=layout).check(hip, dev, "f16", "gelu_tanh")


@pytest.mark.parametrize("tiles", TILES)
def test_tiles_of_extremes_and_scales_that_are_not_finite(hip, dev, tiles):
    """Blocks of the largest quants, a token and two features whose scales are infinite or NaN: theirs alone are
    lost."""
    tokens, wide_ = TILES[tiles]
    c = Case(288, wide_, tokens, seed=10)
    for m, step, quants in ((c.gate, 18, 0x00), (c.up, 18, 0x00), (c.y, 34, 0x80)):
        m.reshape(m.shape[0], -1, step)[::3, ::2, 2:] = quants
    plain_ = c.run(hip, dev, "f32", "relu")[0]
    want, tol = want_of(c.gate, c.up, c.y, "relu", "f32")
    assert (np.abs(plain_ - want) <= tol).all()
    clean = c.run(hip, dev, "f32", "silu")[0].copy()
    inf, nan = (np.array([x], np.uint16).view(np.uint8) for x in (0x7C00, 0x7E00))
    c.y[7, 102:104], c.gate[40, 144:146], c.up[wide_ - 1, 0:2] = inf, nan, inf
    got = c.run(hip, dev, "f32", "silu")[0]
    lost = np.zeros(got.shape, bool)
    lost[7], lost[:, [40, wide_ - 1]] = True, True
    assert not np.isfinite(got[lost]).any()
    assert np.array_equal(got[~lost], clean[~lost])


@pytest.mark.parametrize("tokens,n,wide_", [(1, 64, 70), (6, 64, 70), (500, 64, 4090)])
def test_rows_more_than_32_bits_apart(hip, dev, tokens, n, wide_):
    """Weight rows, rows of activations and of results whose offsets pass 2^32 bytes, the products and their
    blocks what they are side by side."""
    c = Case(n, wide_, tokens, seed=12)
    out, out8 = c.run(hip, dev, "f16", "silu")
    bx = (1 << 33) // wide_ // 2 * 2
    by, step, row8 = ((1 << 33) // tokens // 2 * 2 if tokens > 1 else 0 for _ in range(3))
    by = min(by, 1 << 26)
    bx = min(bx, 1 << 26)

    def apart(rows, stride):
        t = torch.empty(rows.shape[0] * stride + rows.shape[1] if rows.shape[0] > 1 else rows.shape[1],
                        dtype=torch.uint8, device=dev)
        torch.as_strided(t, rows.shape, (stride, 1)).copy_(to_dev(rows, dev))
        return t

    gate, up, y = apart(c.gate, bx), apart(c.up, bx), apart(c.y, by)
    to = torch.empty(max(tokens - 1, 0) * step + wide_, dtype=torch.float16, device=dev)
    to8 = torch.empty(max(tokens - 1, 0) * row8 + wide_ // 32 * 34, dtype=torch.uint8, device=dev)
    hip.gated_q4_0_q8_0("f16", "silu", n, to, step, to8, row8, gate, up, bx, y, by, wide_, tokens)
    assert np.array_equal(wide(torch.as_strided(to, (tokens, wide_), (step, 1)).contiguous()), out)
    got = torch.as_strided(to8, (tokens, wide_ // 32 * 34), (row8, 1)).contiguous()
    assert np.array_equal(from_dev(got), out8)
    del gate, up, y, to, to8, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("tokens", [1, 3, 40, 140])
def test_activations(hip, dev, act, tokens):
    """Of projections a few units wide, and a hundred times that: where the exponential leaves
    float32 both ways."""
    for scale in (1.0, 100.0):
        c = Case(352, 96, tokens, seed=5)
        c.gate = synth.q4_0_matrix(96, 352, 77, scale * 352 ** -0.5)
        c.check(hip, dev, "f32", act)


@pytest.mark.parametrize("tokens", [1, 4, 20, 130])
@pytest.mark.parametrize("apart,layout", [((2, 2), "apart"), ((6, 34), "apart"), ((16, 16), "apart"),
                                          ((0, 0), "in turn")])
def test_strides(hip, dev, tokens, apart, layout):
    c = Case(224, 70, tokens, seed=7, apart=apart, layout=layout)
    for elem in ELEMS:
        c.check(hip, dev, elem, "gelu_tanh")


@pytest.mark.parametrize("tokens", [1, 2, 5, 140])
def test_one_output_or_the_other(hip, dev, tokens):
    """The same bits, where the same order of sums serves both."""
    c = Case(128, 96, tokens, seed=8)
    both = c.run(hip, dev, "f16", "relu")
    assert np.array_equal(c.run(hip, dev, "f16", "relu", q8=False)[0], both[0])
    assert np.array_equal(c.run(hip, dev, "f16", "relu", out=False)[1], both[1])


@pytest.mark.parametrize("tokens", [1, 2, 40, 140])
def test_no_blocks(hip, dev, tokens):
    """n below 32: both projections are 0, and the weights are not looked at."""
    out = torch.full((tokens, 40), 7.0, device=dev)
    q8 = torch.full((tokens, 34), 0xEE, dtype=torch.uint8, device=dev)
    hip.gated_q4_0_q8_0("f32", "silu", 31, out, 40, q8, 34, None, None, 0, None, 0, 40, tokens)
    assert (from_dev(out) == 0.0).all() and (from_dev(q8) == 0).all()


@pytest.mark.parametrize("tokens", [1, 3, 33, 140])
def test_scales_that_are_not_finite(hip, dev, tokens):
    """Of a weight row: its feature is lost for every token; of a token: all of its features."""
    c = Case(96, 70, tokens, seed=9)
    clean = c.run(hip, dev, "f32", "silu")[0].copy()
    bad = np.array([0x7C00], np.uint16).view(np.uint8), np.array([0x7E00], np.uint16).view(np.uint8)
    c.gate[3, 18:20], c.up[40, 0:2], c.up[69, 36:38] = bad[0], bad[1], bad[0]
    if tokens > 1:
        c.y[tokens - 1, 34:36] = bad[0]
    got = c.run(hip, dev, "f32", "silu")[0]
    lost = np.zeros_like(got, bool)
    lost[:, [3, 40, 69]] = True
    if tokens > 1:
        lost[tokens - 1] = True
    assert not np.isfinite(got[lost]).any()
    assert np.array_equal(got[~lost], clean[~lost])


@pytest.mark.parametrize("tokens", [1, 40, 140])
def test_extremes_of_the_blocks(hip, dev, tokens):
    """All quants at their ends and the largest scales: sums of a block of 32 8 128, exact."""
    n, wide_ = 64, 64
    c = Case(n, wide_, tokens, seed=10)
    for m, byte in ((c.gate, 0x00), (c.up, 0xFF)):
        b = m.reshape(wide_, -1, 18)
        b[..., 2:] = byte
        b[..., :2] = np.array([65504.0], np.float16).view(np.uint8)
    y = c.y.reshape(tokens, -1, 34)
    y[..., 2:] = 0x80
    y[..., :2] = np.array([1.0], np.float16).view(np.uint8)
    c.check(hip, dev, "f32", "relu")


def test_same_bits_twice_and_captured(hip, dev):
    for tokens in (1, 24, 200):
        c = Case(512, 160, tokens, seed=11)
        a, b = (c.run(hip, dev, "f32", "silu") for _ in range(2))
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
        dg, du = to_dev(c.gate, dev), to_dev(c.up, dev)
        y = torch.zeros(tokens, 512 // 32 * 34, dtype=torch.uint8, device=dev)
        out = torch.zeros(tokens, 160, device=dev)

        def step():
            hip.gated_q4_0_q8_0("f32", "silu", 512, out, 160, None, 0, dg, du, 288, y, 544, 160,
                                tokens)

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for r in range(3):
            y.copy_(to_dev(c.y if r % 2 == 0 else c.y[::-1].copy(), dev))
            torch.cuda.synchronize()
            graph.replay()
            assert np.array_equal(from_dev(out), a[0] if r % 2 == 0 else a[0][::-1])
            out.zero_()
