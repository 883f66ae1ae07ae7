"""examples/paged_attention.py: its layer against float64, step by step."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import kv_plain
from gpu_util import from_dev

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(__file__), "..", "examples", "paged_attention.py")


@pytest.fixture(scope="module")
def example(hip):
    spec = importlib.util.spec_from_file_location("paged_attention", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def cached(hip, layer, r):
    """Keys and values of request r as the cache holds them, float64."""
    n, ps = int(layer.lengths[r]), layer.page_size
    t = torch.arange(n, device=layer.device)
    slots = layer.block_table[r, t // ps].long() * ps + t % ps
    k, v = (torch.empty((n, layer.kv_heads, layer.dim), device=layer.device) for _ in range(2))
    hip.kv_load_q4_0("f32", layer.cache, layer.pages, ps, slots, k, k.stride(0), k.stride(1), v,
                     v.stride(0), v.stride(1), n, layer.kv_heads, layer.dim)
    return from_dev(k).astype(np.float64), from_dev(v).astype(np.float64)


@pytest.mark.parametrize("window", [0, 40])
def test_layer(hip, dev, example, window):
    layer = example.PagedAttention(hidden=256, heads=6, kv_heads=2, head_dim=64, page_size=16,
                                   pages=40, requests=3, most_tokens=320, window=window)
    rng = np.random.default_rng(3)
    weights = synth_rows(layer.w_out, layer.heads * layer.dim)
    for added in ([37, 0, 16], [1, 5, 1], [1, 1, 1], [0, 130, 1], [1, 1, 1]):
        x = torch.from_numpy(rng.standard_normal((sum(added), 256)).astype(np.float32)).to(dev)
        y = layer.step(x, added)
        q, att = from_dev(layer.last["q"]), from_dev(layer.last["attended"])
        at = 0
        for r, n in enumerate(added):
            k, v = cached(hip, layer, r)
            if not n:
                continue
            rows = q[at:at + n].astype(np.float64)
            want = kv_plain.attend(rows, k, v, int(layer.lengths[r]) - n, 64 ** -0.5, True, window)
            # a score is off by 2^-21 |q||k| / 8 at most, an output by twice that and 2^-20 of the
            # largest value
            qk = np.linalg.norm(rows, axis=-1).max() * np.linalg.norm(k, axis=-1).max() / 8
            tol = 2 * np.abs(v).max() * (2.0 ** -21 * qk + 2.0 ** -20)
            got = att[at:at + n].reshape(n, layer.heads, layer.dim)
            assert np.abs(got - want).max() <= tol
            at += n
        rows8 = synth_rows(example.q8_rows(layer.last["attended"]), layer.heads * layer.dim)
        want = from_dev(x) + rows8 @ weights.T
        # 12 blocks summed in f32, each a few roundings of products below its norms' product
        norms = np.linalg.norm(rows8, axis=-1)[:, None] * np.linalg.norm(weights, axis=-1)[None]
        assert (np.abs(from_dev(y) - want) <= 2.0 ** -19 * (norms + np.abs(want))).all()
    assert layer.lengths.tolist() == [40, 137, 20]
    assert layer.pages_taken == 3 + 9 + 2


def synth_rows(rows, n):
    """Q8_0 rows on the device -> their values, float64."""
    b = from_dev(rows).reshape(-1, 34)
    d = np.ascontiguousarray(b[:, :2]).view(np.float16).astype(np.float64)
    return (b[:, 2:].view(np.int8) * d).reshape(-1, n)


def test_decode_continues_a_prompt(hip, dev, example):
    """A prompt in one step, and the same tokens as a prompt and single tokens: the same cache bytes,
    and outputs that differ by the attention's own rounding."""
    x = torch.randn((50, 1024), generator=torch.Generator().manual_seed(5)).to(dev)
    one = example.PagedAttention(requests=1, pages=8)
    one.step(x, [50])
    whole = one.last["attended"]
    two = example.PagedAttention(requests=1, pages=8)
    two.step(x[:47], [47])
    for i in range(47, 50):
        two.step(x[i:i + 1], [1])
        off = (two.last["attended"] - whole[i:i + 1]).abs().max()
        assert float(off) <= 2.0 ** -17 * float(whole.abs().max())
    for a, b in zip(cached(hip, one, 0), cached(hip, two, 0)):
        assert np.array_equal(a, b)


def test_full_cache(hip, dev, example):
    layer = example.PagedAttention(requests=2, pages=3)
    with pytest.raises(RuntimeError):
        layer.step(torch.zeros((97, 1024), device=dev), [65, 32])
    assert layer.pages_taken == 0
