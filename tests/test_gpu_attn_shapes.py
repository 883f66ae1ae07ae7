"""attn_q4_0 where its work is cut up: decode shared out over work-groups by the requests' lengths,
prompts in parts of the context, and calls that hold both; and prompts whose value scales are not
finite.  Oracle and tolerances: those of test_gpu_kv_cache.Setup (float64)."""
import numpy as np
import pytest

from gpu_util import to_dev
from test_gpu_kv_cache import ELEMS, Setup, wide

pytestmark = pytest.mark.gpu


def ragged(seed, n, most, none=5):
    """n lengths of up to `most`, every none-th 0 or 1; the first the longest."""
    rng = np.random.default_rng(seed)
    got = rng.integers(1, most + 1, n)
    got[none - 1::none] = rng.integers(0, 2, len(got[none - 1::none]))
    got[0] = most
    return [int(x) for x in got]


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("n,most,heads,kv,dim,page", [
    (70, 2500, 4, 2, 64, 16),     # more requests than a wave has lanes
    (150, 1300, 6, 3, 64, 48),
    (33, 2100, 8, 4, 128, 64),
    (20, 2600, 4, 4, 192, 16),
    (20, 2600, 3, 3, 256, 32),
    (3, 700, 40, 2, 64, 16),      # two tiles a request and kv head
    (300, 60, 4, 2, 64, 16),      # a work-group a tile
    (65, 1500, 16, 8, 64, 16),
])
def test_decode_of_ragged_requests(hip, dev, elem, n, most, heads, kv, dim, page):
    lengths = ragged(n, n, most)
    s = Setup(dev, elem, lengths, [1] * n, heads, kv, dim, page, seed=n)
    s.check(hip)
    s.check(hip, window=300)


@pytest.mark.parametrize("elem", ELEMS)
def test_requests_without_new_tokens(hip, dev, elem):
    """Requests that add nothing lie between those that do, whole runs of 64 of them too."""
    n = 210
    added = [1 if r in (0, 3, 64, 200, 209) else 0 for r in range(n)]
    lengths = [700 + 20 * (r % 7) if a or r % 50 == 0 else 3 for r, a in enumerate(added)]
    s = Setup(dev, elem, lengths, added, 8, 4, 64, 16, seed=5)
    s.check(hip)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 150), (False, 0)])
def test_drafted_tokens(hip, dev, elem, causal, window):
    """A few new tokens each, several tiles of rows: the tiles of one request are cut alike."""
    n = 34
    rng = np.random.default_rng(11)
    lengths = [max(x, 4) for x in ragged(6, n, 1400)]
    added = [int(x) for x in rng.integers(0, 5, n)]
    added[0] = 4
    s = Setup(dev, elem, lengths, added, 24, 2, 64, 16, seed=8)  # up to 48 rows a kv head
    s.check(hip, causal=causal, window=window)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("lengths,added,heads,kv,dim", [
    ([2000, 1500, 900, 40], [1, 300, 2, 40], 8, 2, 64),
    ([1300, 700, 0, 5, 1290], [90, 1, 1, 5, 1], 4, 1, 128),
    ([900, 1100], [150, 1], 2, 1, 256),
])
def test_prompts_beside_decode(hip, dev, elem, lengths, added, heads, kv, dim):
    s = Setup(dev, elem, lengths, added, heads, kv, dim, 32, seed=9)
    s.check(hip)
    s.check(hip, causal=False)
    s.check(hip, window=333)


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
def test_prompts_in_parts(hip, dev, elem, dim):
    """One kv head of a chunk on a long context: 8 parts and more of a row."""
    s = Setup(dev, elem, [4500], [20], 2, 1, dim, 16, seed=10)
    s.check(hip)
    s.check(hip, window=1100)


@pytest.mark.parametrize("max_length", [2 ** 20, 2 ** 30])
def test_generous_bounds(hip, dev, max_length):
    """max_length far past the lengths: coarser units where they would not fit 31 bits otherwise."""
    n = 36
    s = Setup(dev, "f16", ragged(7, n, 900), [1] * n, 16, 8, 64, 16, seed=12)
    out = wide(s.run(hip, max_length=max_length))
    want = s.want()
    assert (np.abs(out - want) <= s.tolerance(want)).all()


@pytest.mark.parametrize("elem", ELEMS)
@pytest.mark.parametrize("dim", [64, 192, 256])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_value_scales_that_are_not_finite(hip, dev, elem, dim, bad):
    """In a prompt: rows that see the token are not finite in its block, the others and the other
    blocks are as they were."""
    at, block, length = 70, 1, 131
    s = Setup(dev, elem, [length], [length], 2, 1, dim, 16, seed=13)
    clean = s.run(hip)
    ps = s.page
    page, t = int(s.table[0, at // ps]), at % ps
    lay = s.cache
    o = 2 * lay.quants + lay.scales + ((t // 4) * lay.nb + block) * 8 + (t % 4) * 2
    lay.bytes[page, 0, o:o + 2] = np.array([bad], np.float16).view(np.uint8)
    bufs = list(s.buffers())
    bufs[0] = to_dev(lay.bytes.reshape(-1), dev)
    got, want = wide(s.run(hip, bufs=bufs)), wide(clean)
    hit = slice(32 * block, 32 * block + 32)
    assert not np.isfinite(got[at:, :, hit]).any()
    got[at:, :, hit] = want[at:, :, hit]
    # a step that holds such a scale takes its values by another way: their own rounding at most
    assert (np.abs(got - want) <= 2 * s.tolerance(want)).all()


@pytest.mark.parametrize("elem", ELEMS)
def test_many_prompts(hip, dev, elem):
    """More requests than a wave has lanes, their tiles from none to several."""
    n = 140
    rng = np.random.default_rng(14)
    added = [int(x) for x in rng.integers(0, 60, n)]
    added[::9] = [0] * len(added[::9])
    added[70], added[130] = 150, 1
    lengths = [a + int(x) for a, x in zip(added, rng.integers(0, 120, n))]
    s = Setup(dev, elem, lengths, added, 4, 1, 64, 16, seed=15)
    s.check(hip)
    s.check(hip, window=50)


@pytest.mark.parametrize("requests", [3, 70])
def test_chunks_in_parts_beside_short_ones(hip, dev, requests):
    """Parts by the longest request, which the others have fewer of."""
    lengths = [2100] + [30 + 7 * r for r in range(requests - 1)]
    added = [64] + [20] * (requests - 1)
    s = Setup(dev, "f32", lengths, added, 2, 1, 64, 16, seed=16)
    s.check(hip)
    s.check(hip, causal=False)
