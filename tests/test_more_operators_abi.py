"""Host checks of the norm, the gated product and the drafted tokens' entries: refusals before any launch (the
addresses are made up: nothing may run), empty calls, and what a launch holds."""
import ctypes

import pytest

import launches
import tcrv_hip

A, B, C, D, E, F, G, H, I = (i << 20 for i in range(1, 10))
F32, F16, BF16 = 7, 9, 10
NULL, SIZE, ALIGN, LARGE, UNSUPPORTED, OK = (
    tcrv_hip.ERR_NULL_POINTER, tcrv_hip.ERR_BAD_SIZE, tcrv_hip.ERR_MISALIGNED,
    tcrv_hip.ERR_TOO_LARGE, tcrv_hip.ERR_UNSUPPORTED, tcrv_hip.OK)


def status(name, args, **changed):
    assert set(changed) <= set(args)
    args = dict(args, **changed)
    return tcrv_hip.call(name, *args.values(), 0, check=False)


NORM = dict(elem=F32, x=A, x_token=4096, residual=B, residual_token=4096, sum=C, sum_token=4096,
            weight=D, eps=1e-5, y=E, y_token=4096, q8=F, q8_token=4352, tokens=8, n=4096)


@pytest.mark.parametrize("want,changed", [
    (UNSUPPORTED, dict(elem=8)), (UNSUPPORTED, dict(elem=0)), (SIZE, dict(eps=-1e-9)),
    (SIZE, dict(eps=float("nan"))), (SIZE, dict(eps=float("inf"))), (SIZE, dict(x_token=4095)),
    (SIZE, dict(residual_token=0)), (SIZE, dict(sum_token=1)), (SIZE, dict(y_token=4000)),
    (SIZE, dict(q8_token=4350)), (NULL, dict(x=0)), (NULL, dict(sum=0, y=0, q8=0)),
    (ALIGN, dict(x=A + 2)), (ALIGN, dict(residual=B + 1)), (ALIGN, dict(elem=BF16, sum=C + 1)),
    (ALIGN, dict(y=E + 3)), (ALIGN, dict(weight=D + 2)), (ALIGN, dict(q8=F + 1)),
    (ALIGN, dict(q8_token=4353)), (LARGE, dict(tokens=1 << 24)),
    (LARGE, dict(n=1 << 31, x_token=1 << 31)), (OK, dict(tokens=0)), (OK, dict(n=0)),
    (OK, dict(tokens=0, x=0, sum=0, y=0, q8=0)),
])
def test_norm(want, changed):
    assert status("tcrv_hip_add_rms_norm", NORM, **changed) == want


GATED = dict(elem=F32, act=0, n=4096, out=A, out_token=11008, q8=B, q8_token=11696, gate=C, up=D,
             bx=2304, vy=E, by=4352, nr=11008, nc=3)


@pytest.mark.parametrize("want,changed", [
    (UNSUPPORTED, dict(elem=3)), (UNSUPPORTED, dict(act=4)), (UNSUPPORTED, dict(act=-1)),
    (SIZE, dict(out_token=11007)), (SIZE, dict(q8_token=11694)), (SIZE, dict(bx=2302)),
    (SIZE, dict(by=4350)), (NULL, dict(out=0, q8=0)), (NULL, dict(gate=0)), (NULL, dict(up=0)),
    (NULL, dict(vy=0)), (ALIGN, dict(out=A + 2)), (ALIGN, dict(elem=F16, out=A + 1)),
    (ALIGN, dict(q8=B + 1)), (ALIGN, dict(q8_token=11697)), (ALIGN, dict(gate=C + 1)),
    (ALIGN, dict(up=D + 1)), (ALIGN, dict(vy=E + 1)), (ALIGN, dict(bx=2305)),
    (ALIGN, dict(by=4353)), (LARGE, dict(nr=0x80000000, out_token=1 << 33, q8_token=1 << 33)),
    (LARGE, dict(nc=1 << 24)), (LARGE, dict(n=1 << 36)), (LARGE, dict(bx=(1 << 26) + 2)),
    (LARGE, dict(by=(1 << 26) + 2)), (LARGE, dict(n=1 << 26)), (OK, dict(nr=0)), (OK, dict(nc=0)),
    (OK, dict(nr=0, out=0, q8=0, gate=0, up=0, vy=0)),
])
def test_gated(want, changed):
    assert status("tcrv_hip_gated_q4_0_q8_0", GATED, **changed) == want


TABLES = dict(parents=A, first=B, length=C, requests=4, ancestors=D, words=2, positions=E,
              max_tokens=100)


@pytest.mark.parametrize("want,changed", [
    (NULL, dict(parents=0)), (NULL, dict(first=0)), (NULL, dict(length=0)),
    (NULL, dict(ancestors=0)), (NULL, dict(positions=0)), (ALIGN, dict(ancestors=D + 4)),
    (ALIGN, dict(parents=A + 2)), (ALIGN, dict(first=B + 1)), (ALIGN, dict(length=C + 2)),
    (ALIGN, dict(positions=E + 1)), (SIZE, dict(words=0)), (LARGE, dict(max_tokens=1 << 31)),
    (LARGE, dict(requests=1 << 24)), (LARGE, dict(words=1 << 31)), (OK, dict(max_tokens=0)),
    (OK, dict(max_tokens=0, parents=0, ancestors=0)),
])
def test_tree_tables(want, changed):
    assert status("tcrv_hip_tree_tables", TABLES, **changed) == want


ATTN = dict(elem=F32, q=A, q_token=4096, q_head=128, cache=B, pages=64, page_size=16,
            block_table=C, table_stride=8, first=D, length=D + 4096, ancestors=I, words=1, requests=2,
            tokens=20, max_added=10, max_length=128, heads=32, kv_heads=8, head_dim=128, scale=0.1,
            window=0, out=E, out_token=4096, out_head=128, workspace=F, workspace_bytes=1 << 30)


@pytest.mark.parametrize("want,changed", [
    (UNSUPPORTED, dict(elem=8)), (SIZE, dict(heads=30)), (SIZE, dict(kv_heads=0)),
    (SIZE, dict(head_dim=80)), (SIZE, dict(page_size=8)), (SIZE, dict(q_head=64)),
    (SIZE, dict(out_token=100)), (SIZE, dict(scale=float("nan"))), (SIZE, dict(words=0)),
    (SIZE, dict(max_added=65)), (SIZE, dict(max_added=129, words=2)), (NULL, dict(q=0)),
    (NULL, dict(out=0)), (NULL, dict(cache=0)), (NULL, dict(block_table=0)), (NULL, dict(first=0)),
    (NULL, dict(length=0)), (NULL, dict(ancestors=0)), (ALIGN, dict(ancestors=I + 4)),
    (ALIGN, dict(q=A + 2)), (ALIGN, dict(cache=B + 4)), (ALIGN, dict(block_table=C + 2)),
    (LARGE, dict(requests=1 << 31)), (LARGE, dict(tokens=1 << 31)), (LARGE, dict(max_length=1 << 31)),
    (LARGE, dict(pages=1 << 31)), (SIZE, dict(out_token=64)), (OK, dict(tokens=0)),
    (OK, dict(requests=0)), (OK, dict(max_added=0)),
])
def test_attn_tree(want, changed):
    assert status("tcrv_hip_attn_tree_q4_0", ATTN, **changed) == want


def test_attn_tree_workspace():
    long = dict(max_length=65536, table_stride=4096)
    need = tcrv_hip.attn_tree_q4_0_workspace_bytes("f32", 2, 20, 10, 65536, 32, 8, 128)
    assert need > 0
    assert status("tcrv_hip_attn_tree_q4_0", ATTN, **long, workspace=0) == NULL
    assert status("tcrv_hip_attn_tree_q4_0", ATTN, **long, workspace=F + 4) == ALIGN
    assert status("tcrv_hip_attn_tree_q4_0", ATTN, **long, workspace_bytes=need - 1) == SIZE
    assert tcrv_hip.attn_tree_q4_0_workspace_bytes("f32", 2, 20, 10, 1 << 40, 32, 8, 128) == 0
    assert tcrv_hip.attn_tree_q4_0_workspace_bytes("f32", 2, 20, 0, 4096, 32, 8, 128) == 0


KEEP = dict(cache=A, pages=64, page_size=16, block_table=B, table_stride=8, first=C, length=D,
            path=E, path_stride=10, count=F, requests=3, max_added=10, kv_heads=8, head_dim=128)


@pytest.mark.parametrize("want,changed", [
    (SIZE, dict(page_size=24)), (SIZE, dict(kv_heads=0)), (SIZE, dict(head_dim=96)),
    (NULL, dict(cache=0)), (NULL, dict(block_table=0)), (NULL, dict(first=0)), (NULL, dict(length=0)),
    (NULL, dict(path=0)), (NULL, dict(count=0)), (ALIGN, dict(cache=A + 8)), (ALIGN, dict(path=E + 2)),
    (ALIGN, dict(count=F + 1)), (ALIGN, dict(first=C + 2)), (ALIGN, dict(length=D + 2)),
    (ALIGN, dict(block_table=B + 2)), (LARGE, dict(requests=1 << 24)), (LARGE, dict(pages=1 << 31)),
    (LARGE, dict(max_added=1 << 31)), (LARGE, dict(table_stride=1 << 31)), (OK, dict(requests=0)),
    (OK, dict(max_added=0)), (OK, dict(path_stride=0)), (OK, dict(pages=0, cache=0)),
])
def test_keep(want, changed):
    assert status("tcrv_hip_kv_keep_q4_0", KEEP, **changed) == want


def test_floats_reach_the_library():
    """The double and float arguments' types: a wrong one would be read from another register."""
    assert tcrv_hip.SIGNATURES["tcrv_hip_add_rms_norm"][8] is ctypes.c_double
    assert tcrv_hip.SIGNATURES["tcrv_hip_attn_tree_q4_0"][20] is ctypes.c_float


@pytest.mark.parametrize("nr,nc,want", [
    (14336, (1 << 24) - 1, LARGE), (8064, (1 << 24) - 1, OK), (8065, (1 << 24) - 1, LARGE),
    (1 << 14, ((1 << 23) - 1) // 128 * 128, OK), (1 << 14, (1 << 23) - 127, LARGE), (0x3fffffc, 1920, OK),
    (0x3fffffc, 2049, LARGE), (0x3fffffc, 64, OK), (192, (1 << 24) - 1, OK), (129, (1 << 24) - 1, OK),
    (96, (1 << 24) - 1, OK),
])
@pytest.mark.parametrize("q8", [False, True])
def test_gated_tiles_that_a_launch_holds(nr, nc, want, q8):
    """Less than 2^23 tiles of 128 x 128, whichever kernel serves the call."""
    assert (-(-nr // 128) * -(-nc // 128) < 1 << 23) == (want == OK)
    (got, made), = launches.replay([("tcrv_hip_gated_q4_0_q8_0", (
        9, 0, 64, P, nr, Q if q8 else 0, nr // 32 * 34, R, S, 36, T, 68, nr, nc))])
    assert got == want and bool(made) == (want == OK)
    assert all(g * b < 1 << 32 for x in made for g, b in zip(x.grid, x.block))


MOST = (1 << 24) - 1
P, Q, R, S, T, U, V, W = ((i + 1) << 50 for i in range(8))


def norm(tokens, n):
    return "tcrv_hip_add_rms_norm", (9, P, n, Q, n, R, n, S, 1e-5, T, n, U, n // 32 * 34, tokens, n)


def gated(nr, nc):
    return "tcrv_hip_gated_q4_0_q8_0", (9, 0, 64, P, nr, Q, nr // 32 * 34, R, S, 36, T, 68, nr, nc)


def attn(requests, tokens, added, length=16, heads=1, kv=1, dim=64):
    return "tcrv_hip_attn_tree_q4_0", (9, P, heads * dim, dim, Q, 64, 16, R, 8, S, T, W, 1 << 20,
                                       requests, tokens, added, length, heads, kv, dim, 0.1, 0, U,
                                       heads * dim, dim, V, 1 << 60)


@pytest.mark.parametrize("call,want", [
    (norm(MOST, 4096), OK), (norm(MOST, 64), OK), (norm(MOST, 1 << 20), OK),
    (gated(64, MOST), OK), (gated(32, MOST), OK), (gated(1, MOST), OK), (gated(0x3fffffc, 1), OK), (gated(0x3fffffc, 5), OK),
    (gated(0x3fffffc, MOST), LARGE), (gated(0x3fffffd, 1), LARGE),
    (("tcrv_hip_tree_tables", (P, Q, R, MOST - 1, S, 1, T, 0x7fffffff)), OK),
    (("tcrv_hip_kv_keep_q4_0", (P, 64, 16, Q, 8, R, S, T, 8, U, MOST, 8, 65535, 64)), OK),
    (attn(MOST, MOST, 1), OK), (attn(MOST + 1, MOST + 1, 1), LARGE),
    (attn(1 << 20, 1 << 20, 1, heads=16, kv=16), LARGE),
    (attn(1, MOST, MOST, heads=1), OK), (attn(1, MOST, MOST, heads=127, kv=127), OK),
    (attn(1, MOST, MOST, heads=128, kv=128), LARGE),
])
def test_most_that_a_launch_holds(call, want):
    (got, made), = launches.replay([call])
    assert got == want
    assert bool(made) == (want == OK)
    for x in made:
        assert all(g * b < 1 << 32 for g, b in zip(x.grid, x.block)), made
        assert all(g <= 65535 for g in x.grid[1:]), made
