"""add_rms_norm on the GPU against its formula: the mean of the squares in float64, everything after it as
single float32 operations.  The root rounds to the same float32 whatever the order of the sum (its terms are
exact in float64, the sum off by 2^-50 of itself, a float32 step 2^-24), so outputs are compared bit by bit."""
import numpy as np
import pytest
import torch

import kv_plain
import synth
from gpu_util import from_dev, to_dev
from test_gpu_kv_cache import ELEMS, TORCH, dev_rows, wide

pytestmark = pytest.mark.gpu

EPS = 1e-5


def plain(x, residual, weight, eps=EPS):
    """(sum, norm) float32 of float32 rows."""
    h = x if residual is None else (x + residual).astype(np.float32)
    with np.errstate(all="ignore"):
        mean = (h.astype(np.float64) ** 2).mean(-1, keepdims=True)
        c = (1.0 / np.sqrt(mean + eps)).astype(np.float32)
        y = (h * c).astype(np.float32)
        return h, y if weight is None else (y * weight).astype(np.float32)


def padded(rows, n, stride, elem, dev, fill=7.0):
    t = torch.full((rows * stride + 8,), fill, dtype=TORCH[elem], device=dev)
    return t


def rows_of(t, off, rows, n, stride):
    return wide(t)[off:off + rows * stride].reshape(rows, stride)[:, :n] if rows else None


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("tokens,n,pad,off", [
    (1, 1, 0, 0), (3, 2, 0, 0), (1, 32, 0, 0), (5, 31, 1, 0), (2, 33, 3, 1), (7, 64, 4, 0),
    (9, 96, 0, 2), (4, 1000, 0, 0), (5, 1024, 32, 0), (3, 1025, 0, 0), (2, 1056, 0, 0),
    (3, 4096, 0, 0), (1, 4096, 0, 1), (2, 4100, 0, 0), (2, 5120, 4, 0), (1, 16384, 0, 0),
    (2, 16385, 0, 0), (2, 16416, 0, 0), (1, 40000, 0, 0), (1027, 64, 0, 0), (300, 320, 0, 0),
    # many rows, of fewer lanes or registers each than a few rows take
    (535, 300, 0, 0), (530, 512, 0, 0), (531, 800, 0, 0), (513, 1600, 0, 0), (521, 4096, 0, 0),
    (514, 8192, 0, 0), (601, 35, 1, 1), (602, 301, 3, 1), (603, 1001, 0, 0), (513, 2001, 0, 0),
    (515, 4001, 1, 3), (47, 128, 0, 0), (33, 256, 8, 0),
])
def test_sum_norm_and_blocks(hip, dev, elem, tokens, n, pad, off):
    rng = np.random.default_rng(tokens * 100003 + n)
    x, residual = (kv_plain.round_to(s * rng.standard_normal((tokens, n)), elem) for s in (0.3, 3.0))
    weight = (1.0 + 0.2 * rng.standard_normal(n)).astype(np.float32)
    h, y = plain(x, residual, weight)
    nb, stride = n // 32, n + pad
    want8 = synth.quantize_q8_0(y[:, :nb * 32]).reshape(tokens, nb * 34) if nb else None
    src = [padded(tokens, n, stride, elem, dev) for _ in range(2)]
    for t, v in zip(src, (x, residual)):
        t[off:off + tokens * stride].view(tokens, stride)[:, :n] = dev_rows(v, elem, dev)
    dw = to_dev(weight, dev)
    for q8_pad in (0, 2):
        out = [padded(tokens, n, stride, elem, dev) for _ in range(2)]
        row8 = nb * 34 + q8_pad
        q8 = torch.full((tokens * row8 + 32,), 0xEE, dtype=torch.uint8, device=dev)
        hip.add_rms_norm(elem, src[0][off:], stride, src[1][off:], stride, out[0][off:], stride, dw,
                         EPS, out[1][off:], stride, q8, row8, tokens, n)
        for t, want in zip(out, (h, y)):
            got = wide(t)
            rows = got[off:off + tokens * stride].reshape(tokens, stride)
            assert np.array_equal(rows[:, :n].view(np.uint32), kv_plain.round_to(want, elem).view(np.uint32))
            assert (rows[:, n:] == 7.0).all() and (got[:off] == 7.0).all()
            assert (got[off + tokens * stride:] == 7.0).all()
        got8 = from_dev(q8)
        rows = got8[:tokens * row8].reshape(tokens, row8)
        if nb:
            assert np.array_equal(rows[:, :nb * 34], want8)
        assert (rows[:, nb * 34:] == 0xEE).all() and (got8[tokens * row8:] == 0xEE).all()


@pytest.mark.parametrize("n", [96, 4096, 16384, 20000])
@pytest.mark.parametrize("what", ["sum", "y", "q8", "no residual", "no weight"])
def test_outputs_and_inputs_that_are_left_out(hip, dev, n, what):
    tokens = 3
    rng = np.random.default_rng(n)
    x, residual = (rng.standard_normal((tokens, n)).astype(np.float32) for _ in range(2))
    weight = rng.standard_normal(n).astype(np.float32)
    h, y = plain(x, None if what == "no residual" else residual,
                 None if what == "no weight" else weight)
    dx, dr, dw = (to_dev(v, dev) for v in (x, residual, weight))
    both = what.startswith("no")
    total = torch.zeros(tokens, n, device=dev) if what == "sum" or both else None
    out = torch.zeros(tokens, n, device=dev) if what == "y" or both else None
    q8 = torch.zeros(tokens, n // 32 * 34, dtype=torch.uint8, device=dev) if what == "q8" else None
    hip.add_rms_norm("f32", dx, n, None if what == "no residual" else dr, n, total, n,
                     None if what == "no weight" else dw, EPS, out, n, q8, n // 32 * 34, tokens, n)
    if total is not None:
        assert np.array_equal(from_dev(total), h)
    if out is not None:
        assert np.array_equal(from_dev(out), y)
    if q8 is not None:
        assert np.array_equal(from_dev(q8).reshape(-1), synth.quantize_q8_0(y))


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("n", [64, 4096, 16384, 20000])
def test_in_place(hip, dev, elem, n):
    """The stream of residuals takes the sum in its own place, the norm that of x."""
    tokens = 5
    rng = np.random.default_rng(n + 1)
    x, residual = (kv_plain.round_to(rng.standard_normal((tokens, n)), elem) for _ in range(2))
    h, y = plain(x, residual, None)
    for place in ("residual", "x"):
        dx, dr = dev_rows(x, elem, dev), dev_rows(residual, elem, dev)
        total, out = (dr, dx) if place == "residual" else (dx, dr)
        hip.add_rms_norm(elem, dx, n, dr, n, total, n, None, EPS, out, n, None, 0, tokens, n)
        assert np.array_equal(wide(total), kv_plain.round_to(h, elem))
        assert np.array_equal(wide(out), kv_plain.round_to(y, elem))


@pytest.mark.parametrize("off", [0, 2, 8])
@pytest.mark.parametrize("elem,n,row8", [
    ("f32", 32, 48), ("f32", 33, 48), ("f32", 64, 80), ("f32", 64, 96), ("f32", 64, 72), ("f32", 62, 48),
    ("f16", 128, 144), ("bf16", 128, 160), ("f16", 128, 152), ("f16", 124, 112), ("bf16", 64, 80),
    ("f32", 192, 208), ("f16", 512, 560),
])
def test_blocks_of_short_rows_at_other_strides(hip, dev, elem, n, row8, off):
    """Rows of heads, sixteen a work-group, whose blocks begin at places of 16 and 8 bytes and others that are
    not those of dense rows; what lies between them stays."""
    tokens, nb = 37, n // 32
    rng = np.random.default_rng(n + row8)
    x = kv_plain.round_to(rng.standard_normal((tokens, n)), elem)
    want = synth.quantize_q8_0(plain(x, None, None)[1][:, :nb * 32]).reshape(tokens, nb * 34)
    q8 = torch.full((off + tokens * row8 + 32,), 0xEE, dtype=torch.uint8, device=dev)
    assert q8.data_ptr() % 16 == 0
    hip.add_rms_norm(elem, dev_rows(x, elem, dev), n, None, 0, None, 0, None, EPS, None, 0, q8[off:], row8,
                     tokens, n)
    got = from_dev(q8)
    rows = got[off:off + tokens * row8].reshape(tokens, row8)
    assert np.array_equal(rows[:, :nb * 34], want)
    assert (rows[:, nb * 34:] == 0xEE).all() and (got[:off] == 0xEE).all()
    assert (got[off + tokens * row8:] == 0xEE).all()


def test_values_at_the_ends(hip, dev):
    """Rows of zeros (with and without eps), of values whose squares leave float32 both ways, and rows
    that hold an infinity or a NaN: those alone are lost."""
    n = 128
    rng = np.random.default_rng(9)
    x = rng.standard_normal((8, n)).astype(np.float32)
    x[0] = 0.0
    x[1] *= np.float32(1e30)
    x[2] *= np.float32(1e-30)
    x[3, 5] = np.inf
    x[4, 7] = np.nan
    for eps in (0.0, 1e-5, 1e-40):
        h, want = plain(x, None, None, eps)
        out = torch.zeros(8, n, device=dev)
        hip.add_rms_norm("f32", to_dev(x, dev), n, None, 0, None, 0, None, eps, out, n, None, 0, 8, n)
        got = from_dev(out)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
        assert np.isfinite(got[[1, 2, 5, 6, 7]]).all()


def test_captured_and_replayed(hip, dev):
    n, tokens = 4096, 9
    rng = np.random.default_rng(4)
    x, r = (torch.zeros(tokens, n, device=dev) for _ in range(2))
    total, q8 = torch.zeros_like(x), torch.zeros(tokens, n // 32 * 34, dtype=torch.uint8, device=dev)

    def step():
        hip.add_rms_norm("f32", x, n, r, n, total, n, None, EPS, None, 0, q8, n // 32 * 34, tokens, n)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(3):
        a, b = (rng.standard_normal((tokens, n)).astype(np.float32) for _ in range(2))
        x.copy_(to_dev(a, dev))
        r.copy_(to_dev(b, dev))
        torch.cuda.synchronize()
        graph.replay()
        h, y = plain(a, b, None)
        assert np.array_equal(from_dev(total), h)
        assert np.array_equal(from_dev(q8).reshape(-1), synth.quantize_q8_0(y))


def test_rows_more_than_32_bits_apart(hip, dev):
    n, tokens, stride = 1000, 300, 1 << 23
    rng = np.random.default_rng(8)
    x, r = (kv_plain.round_to(rng.standard_normal((tokens, n)), "f16") for _ in range(2))
    h, y = plain(x, r, None)
    far = [torch.empty((tokens - 1) * stride + n, dtype=torch.float16, device=dev) for _ in range(4)]
    rows = [torch.as_strided(t, (tokens, n), (stride, 1)) for t in far]
    for t, v in zip(rows, (x, r)):
        t.copy_(dev_rows(v, "f16", dev))
    row8 = 1 << 24
    q8 = torch.empty((tokens - 1) * row8 + 31 * 34, dtype=torch.uint8, device=dev)
    hip.add_rms_norm("f16", far[0], stride, far[1], stride, far[2], stride, None, EPS, far[3], stride, q8,
                     row8, tokens, n)
    for t, want in zip(rows[2:], (h, y)):
        assert np.array_equal(wide(t.contiguous()), kv_plain.round_to(want, "f16"))
    got = torch.as_strided(q8, (tokens, 31 * 34), (row8, 1)).contiguous()
    assert np.array_equal(from_dev(got).reshape(-1), synth.quantize_q8_0(np.ascontiguousarray(y[:, :992])))
    del far, rows, q8, got
    torch.cuda.empty_cache()
