"""Which kernels the norm, the gated products and the attention over trees launch at a size, and their grids,
replayed without a GPU (tests/launches.py)."""
import re

import pytest

import launches
import tcrv_hip

A, B, C, D, E, F, G, H = ((k + 1) << 40 for k in range(8))
KERNEL = r"(add_rms_norm_rows|gated_one|gated_spans|gated_tiles|attn_q4_0_(?:rows16|tiles|join_few|join))"


def run(call):
    status, made = launches.replay([call])[0]
    assert status == 0
    return [(re.search(KERNEL, x.name)[1], x.grid[0], x.block[0]) for x in made]


def norm(elem, tokens, n, pad=0):
    return "tcrv_hip_add_rms_norm", (tcrv_hip.FLOAT_ELEM[elem], A, n + pad, B, n + pad, C, n + pad, D,
                                     1e-5, E, n + pad, F, n // 32 * 34, tokens, n)


@pytest.mark.parametrize("args,want", [
    # heads' rows: 16 a work-group
    (("f16", 60000, 128), (3750, 256)), (("f32", 1, 256), (1, 256)), (("f16", 4096, 512), (256, 256)),
    (("f32", 4096, 257), (1024, 256)),
    # a few long rows, on as many threads as a work-group has
    (("f32", 1, 4096), (1, 1024)), (("f16", 256, 8192), (256, 1024)), (("f32", 512, 4096), (512, 1024)), (("f16", 257, 8192), (257, 256)), (("f32", 3, 1024), (3, 1024)),
    # many: four, or one, a work-group
    (("f16", 257, 1024), (65, 256)), (("f32", 4096, 1024), (1024, 256)), (("f16", 4096, 4096), (4096, 256)),
    (("f32", 4096, 4096), (4096, 256)), (("f32", 4096, 4100), (4096, 1024)),
    # past a row's registers
    (("f32", 2, 16388), (2, 1024)), (("f16", 1000, 40000), (1000, 1024)),
])
def test_rows_of_the_norm(args, want):
    (name, grid, block), = run(norm(*args))
    assert (grid, block) == want


def gated(tokens, n, wide, q8=False, elem="f32"):
    return "tcrv_hip_gated_q4_0_q8_0", (tcrv_hip.FLOAT_ELEM[elem], 0, n, A, wide, B if q8 else 0,
                                        wide // 32 * 34, C, D, n // 32 * 18, E, n // 32 * 34, wide,
                                        tokens)


@pytest.mark.parametrize("args,want", [
    ((1, 4096, 11008), ("gated_one", 2752, 256)), ((1, 4096, 11008, True), ("gated_one", 344, 1024)),
    ((1, 32, 33), ("gated_one", 9, 256)), ((1, 32, 33, True), ("gated_one", 2, 1024)),
    ((2, 4096, 11008), ("gated_one", 2752, 256)), ((2, 4096, 11008, True), ("gated_one", 344, 1024)),
    ((4, 4096, 11008), ("gated_one", 2752, 256)), ((3, 4096, 11008, True), ("gated_spans", 344, 512)),
    ((4, 4096, 14336), ("gated_spans", 448, 512)), ((5, 4096, 11008), ("gated_spans", 344, 512)),
    # 16 features a work-group
    ((5, 4096, 4096), ("gated_spans", 256, 512)), ((5, 4096, 4097), ("gated_spans", 129, 512)),
    ((64, 4096, 2048), ("gated_spans", 256, 512)), ((64, 4096, 4096, True), ("gated_spans", 256, 512)), ((64, 4096, 11008), ("gated_spans", 688, 512)),
    ((128, 4096, 14336), ("gated_tiles", 224, 512)), ((512, 4096, 14336), ("gated_tiles", 448, 512)),
    ((2048, 4096, 14336), ("gated_tiles", 1792, 512)), ((2048, 64, 96), ("gated_spans", 192, 512)),
    # tiles of 64 and of 128 features, of tests/test_gpu_gated.py
    ((500, 32, 4090), ("gated_tiles", 64 * 4, 512)), ((630, 32, 4590), ("gated_tiles", 36 * 5, 512)),
])
def test_kernel_of_the_products(args, want):
    assert run(gated(*args)) == [want]


def tree(elem, requests, tokens, nodes, length, heads, kv, dim, window=0):
    return "tcrv_hip_attn_tree_q4_0", (
        tcrv_hip.FLOAT_ELEM[elem], A, heads * dim, dim, B, 1 << 20, 16, C, 1 << 16, D, E, F,
        -(-nodes // 64), requests, tokens, nodes, length, heads, kv, dim, dim ** -0.5, window, G,
        heads * dim, dim, H, 1 << 50)


@pytest.mark.parametrize("args,want", [
    # up to 64 rows a kv head go on the tiles of few rows, whatever the requests
    (("f32", 1, 7, 7, 538, 32, 8, 128), ["rows16", "join_few"]),
    (("f16", 4, 64, 16, 100, 32, 8, 128), ["rows16"]),
    (("f16", 64, 512, 8, 4104, 32, 8, 128), ["rows16", "join_few"]),
    (("bf16", 1, 16, 16, 20, 8, 2, 64), ["rows16"]),
    # more rows on those of prompts
    (("f16", 6, 384, 64, 8256, 32, 8, 128), ["tiles", "join"]),
    (("f16", 200, 200 * 64, 64, 600, 32, 8, 128), ["tiles"]),
])
def test_kernels_of_trees(args, want):
    got = [name.replace("attn_q4_0_", "") for name, _, _ in run(tree(*args))]
    assert got == want


@pytest.mark.parametrize("elem", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [700, 3000])
@pytest.mark.parametrize("cached,nodes,heads,kv,dim,want", [
    # the sizes of test_gpu_tree.py whose tiles are in parts, which a join brings together
    ([4100, 300, 2500], [200, 70, 130], 8, 2, 64, ["rows16", "join_few", "tiles", "join"]),
    ([3500, 5000], [200, 3], 8, 2, 128, ["rows16", "join_few", "tiles", "join"]),
    ([2900], [330], 4, 2, 192, ["tiles", "join"]),
    ([3300], [150], 8, 2, 256, ["tiles", "join"]),
    ([5000, 4100, 90], [16, 9, 16], 8, 2, 128, ["rows16", "join_few"]),
    ([6000], [61], 2, 2, 64, ["rows16", "join_few"]),
    ([3900, 800], [12, 16], 4, 1, 256, ["rows16", "join_few"]),
])
def test_windowed_trees_in_parts(elem, window, cached, nodes, heads, kv, dim, want):
    length = max(c + n for c, n in zip(cached, nodes))
    got = run(tree(elem, len(nodes), sum(nodes), max(nodes), length, heads, kv, dim, window))
    assert [name.replace("attn_q4_0_", "") for name, _, _ in got] == want


@pytest.mark.parametrize("nodes", [1, 16, 17, 200])
@pytest.mark.parametrize("length", [210, 4000, 131072, 1 << 30])
def test_workspace_of_trees_serves_every_window(nodes, length):
    for requests, heads, kv, dim in ((1, 32, 8, 128), (64, 32, 8, 128), (5, 14, 2, 64), (3, 16, 4, 256)):
        tokens = requests * nodes
        need = tcrv_hip.attn_tree_q4_0_workspace_bytes("f16", requests, tokens, nodes, length, heads, kv,
                                                       dim)
        calls = []
        for window in (0, 1, 100, 5000, 1 << 40):
            name, args = tree("f16", requests, tokens, nodes, length, heads, kv, dim, window)
            calls.append((name, args[:-1] + (need,)))
        assert all(status == 0 for status, _ in launches.replay(calls))


def test_every_kernel_is_reached():
    """No instantiation that no call launches."""
    calls = []
    for elem in ("f32", "f16", "bf16"):
        for tokens in (1, 2, 4, 5, 128, 2048):
            for n, wide, q8 in ((32, 4096, False), (32, 4096, True), (4096, 4096, False),
                                (4096, 14336, True)):
                calls.append(gated(tokens, n, wide, q8, elem))
        for tokens in (3, 2000):
            # whole groups of 8 and of 4 values, and others
            for n in (64, 256, 512, 1024, 2048, 4096, 8192, 16384, 32768, 65536):
                calls += [norm(elem, tokens, n + more) for more in (0, -4, -1)]
        for dim in (64, 128, 192, 256):
            for nodes in (4, 200):
                calls.append(tree(elem, 2, 2 * nodes, nodes, 6000, 8, 1, dim))
    calls += [("tcrv_hip_tree_tables", (A, B, C, 4, D, 2, E, 100)),
              ("tcrv_hip_kv_keep_q4_0", (A, 64, 16, B, 8, C, D, E, 10, F, 3, 10, 8, 128))]
    made = {x.name for _, xs in launches.replay(calls) for x in xs}
    # names with _Float16 among their arguments stay as the compiler writes them
    mine = (r"add_rms_norm_rows|gated_(one|spans|tiles)|tree_tables|kv_keep_q4_0"
            r"|attn_q4_0_(rows16|tiles)(<.*true>|I.*Lb1E)")
    held = {name for name in launches.registered() if re.search(mine, name)}
    assert len(held) > 100 and not held - made, sorted(held - made)
