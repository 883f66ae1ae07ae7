"""examples/drafted_layer.py: its layer's stages against float64, and a kept path's cache against that of
the same tokens one by one."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from gpu_util import from_dev
from test_gpu_example_paged import cached, synth_rows
from test_gpu_gated import want_of

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(__file__), "..", "examples", "drafted_layer.py")


@pytest.fixture(scope="module")
def example(hip):
    spec = importlib.util.spec_from_file_location("drafted_layer", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def path_to(tree, i):
    got = []
    while i >= 0:
        got.insert(0, i)
        i = tree[i]
    return got


def attended_want(layer, r, tree, k, v, q):
    """Request r's nodes over the cached tokens and their ancestors, in float64; k and v of all places."""
    context, share = len(k) - len(tree), layer.heads // layer.kv_heads
    out = np.zeros(q.shape)
    for i in range(len(tree)):
        path = path_to(tree, i)
        low = max(0, context + len(path) - layer.window) if layer.window else 0
        seen = list(range(min(low, context), context))
        seen += [context + j for d, j in enumerate(path) if context + d >= low]
        for h in range(layer.heads):
            z = layer.dim ** -0.5 * (k[seen, h // share] @ q[i, h])
            w = np.exp(z - z.max())
            out[i, h] = w @ v[seen, h // share] / w.sum()
    return out


def blocks_off(y, off):
    """What Q8_0 blocks of rows that are off by `off` at most may differ from y: half a quant, the scale's
    half step in fp16 (2^-11 of up to 127 quants, and 2^-25 of a subnormal one)."""
    top = (np.abs(y) + off).reshape(y.shape[0], -1, 32).max(-1, keepdims=True)
    d = np.broadcast_to(top / 127, (*top.shape[:2], 32)).reshape(y.shape)
    return off + d * (0.5 + 127 * 2.0 ** -11) * (1 + 2.0 ** -20) + 127 * 2.0 ** -25


@pytest.mark.parametrize("window", [0, 40])
def test_stages(hip, dev, example, window):
    layer = example.DraftedLayer(hidden=256, wide=416, heads=6, kv_heads=2, head_dim=64, page_size=16,
                                 pages=48, requests=3, most_tokens=320, window=window)
    rng = np.random.default_rng(3)
    w_out, w_down = synth_rows(layer.w_out, 384), synth_rows(layer.w_down, 416)
    gate, up, scale = from_dev(layer.gate), from_dev(layer.up), from_dev(layer.norm_out).astype(np.float64)
    for added in ([37, 0, 16], [9, 4, 1], [1, 17, 70], [1, 1, 1], [0, 30, 5]):
        trees = None if added[0] == 37 else [example.random_tree(rng, n) for n in added]
        x = torch.from_numpy(rng.standard_normal((sum(added), 256)).astype(np.float32)).to(dev)
        y = from_dev(layer.step(x, added, trees)).astype(np.float64)
        last = {k: from_dev(t) for k, t in layer.last.items() if k != "added"}
        # attention, as the layer without trees: a score is off by 2^-21 |q||k| / 8 at most, an output
        # by twice that and 2^-20 of the largest value
        at = 0
        for r, n in enumerate(added):
            k, v = cached(hip, layer, r)
            if not n:
                continue
            q = last["q"][at:at + n].astype(np.float64)
            tree = list(range(-1, n - 1)) if trees is None else trees[r]
            want = attended_want(layer, r, tree, k, v, q)
            qk = np.linalg.norm(q, axis=-1).max() * np.linalg.norm(k, axis=-1).max() / 8
            tol = 2 * np.abs(v).max() * (2.0 ** -21 * qk + 2.0 ** -20)
            assert np.abs(last["attended"][at:at + n].reshape(want.shape) - want).max() <= tol
            at += n
        # products of 12 and 13 blocks summed in f32, each a few roundings of terms below its norms' product
        rows8 = synth_rows(example.q8_rows(layer.last["attended"]), 384)
        norms = np.linalg.norm(rows8, axis=-1)[:, None] * np.linalg.norm(w_out, axis=-1)[None]
        want = from_dev(x) + rows8 @ w_out.T
        total = last["total"].astype(np.float64)
        assert (np.abs(total - want) <= 2.0 ** -19 * (norms + np.abs(want))).all()
        # the norm is that of the rounded sum but for its roundings: half a step each of the sum, c and two
        # products, and c itself of a mean that moves by at most a step
        want = total / np.sqrt((total ** 2).mean(-1, keepdims=True) + example.EPS) * scale
        assert (np.abs(synth_rows(layer.last["rows"], 256) - want)
                <= blocks_off(want, 8 * 2.0 ** -24 * np.abs(want))).all()
        want, off = want_of(gate, up, last["rows"], "silu", "f32")
        assert (np.abs(synth_rows(layer.last["inner"], 416) - want) <= blocks_off(want, off)).all()
        inner = synth_rows(layer.last["inner"], 416)
        norms = np.linalg.norm(inner, axis=-1)[:, None] * np.linalg.norm(w_down, axis=-1)[None]
        want = total + inner @ w_down.T
        assert (np.abs(y - want) <= 2.0 ** -19 * (norms + np.abs(want))).all()
        if trees is not None:
            layer.keep([path_to(t, n - 1) for t, n in zip(trees, added)])
    assert len(layer.free) == 48 - int((-(-layer.lengths // 16)).sum())


def test_kept_paths_are_those_tokens_one_by_one(hip, dev, example):
    """After each step the cache of the accepted paths is, bit for bit, that of a layer which was given the
    paths' tokens one at a time, and the pages that are left are no page of a table twice."""
    rng, gen = np.random.default_rng(7), torch.Generator().manual_seed(5)
    most = dict(requests=2, pages=24, page_size=16, most_tokens=256)
    drafted, single = example.DraftedLayer(**most), example.DraftedLayer(**most)
    x = torch.randn((47 + 14, 1024), generator=gen).to(dev)
    drafted.step(x, [47, 14])
    single.step(x, [47, 14])
    for nodes in ([20, 5], [3, 40], [17, 0], [1, 1], [33, 9]):
        trees = [example.random_tree(rng, n) for n in nodes]
        x = torch.randn((sum(nodes), 1024), generator=gen).to(dev)
        drafted.step(x, nodes, trees)
        paths = [path_to(t, int(rng.integers(-1, n))) if n else [] for t, n in zip(trees, nodes)]
        drafted.keep(paths)
        begin = [0, nodes[0]]
        for r in range(2):
            for node in paths[r]:
                single.step(x[begin[r] + node:begin[r] + node + 1], [r == 0, r == 1])
        assert drafted.lengths.tolist() == single.lengths.tolist()
        assert from_dev(drafted.context).tolist() == drafted.lengths.tolist()
        for r in range(2):
            for a, b in zip(cached(hip, drafted, r), cached(hip, single, r)):
                assert np.array_equal(a, b)
        table = from_dev(drafted.block_table)
        used = [p for r in range(2) for p in table[r, :-(-int(drafted.lengths[r]) // 16)]]
        assert sorted(used + from_dev(drafted.free).tolist()) == list(range(24))


def test_full_cache(hip, dev, example):
    layer = example.DraftedLayer(requests=2, pages=3)
    with pytest.raises(RuntimeError):
        layer.step(torch.zeros((97, 1024), device=dev), [65, 32])
    assert len(layer.free) == 3


def test_main(hip, dev, example, capsys):
    example.main()
    assert "us a step" in capsys.readouterr().out
