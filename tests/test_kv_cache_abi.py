"""Host checks of the paged Q4_0 cache's entries: refusals before any launch (the addresses are
made up: nothing may run), empty calls, sizes."""
import ctypes

import pytest

import tcrv_hip

Q, K, V, CACHE, TABLE, IDS, OUT, WS = (i << 20 for i in range(1, 9))
F32, F16, BF16 = 7, 9, 10
NULL, SIZE, ALIGN, LARGE, UNSUPPORTED, OK = (
    tcrv_hip.ERR_NULL_POINTER, tcrv_hip.ERR_BAD_SIZE, tcrv_hip.ERR_MISALIGNED,
    tcrv_hip.ERR_TOO_LARGE, tcrv_hip.ERR_UNSUPPORTED, tcrv_hip.OK)


def status(name, args, **changed):
    args = dict(args, **changed)
    return tcrv_hip.call(name, *args.values(), 0, check=False)


ROPE_TABLE = dict(scaling=3, n_dims=128, base=10000.0, factor=4.0, trained=4096.0, beta_fast=32.0,
                  beta_slow=1.0, amplitude=0.0, divisors=0, first=0, count=16, table=TABLE)


@pytest.mark.parametrize("want,changed", [
    (UNSUPPORTED, dict(scaling=4)), (UNSUPPORTED, dict(scaling=-1)),
    (SIZE, dict(n_dims=127)), (SIZE, dict(n_dims=0)), (SIZE, dict(base=0.0)),
    (SIZE, dict(base=float("nan"))), (SIZE, dict(base=float("inf"))), (SIZE, dict(base=1.0)),
    (SIZE, dict(factor=-1.0)), (SIZE, dict(factor=float("nan"))), (SIZE, dict(trained=0.0)),
    (SIZE, dict(beta_slow=33.0)), (SIZE, dict(beta_slow=0.0)), (SIZE, dict(amplitude=-1.0)),
    (SIZE, dict(amplitude=float("nan"))), (SIZE, dict(scaling=2, n_dims=2)),
    (NULL, dict(table=0)), (ALIGN, dict(table=TABLE + 4)), (ALIGN, dict(divisors=TABLE + 2)),
    (LARGE, dict(count=1 << 40)), (LARGE, dict(first=1 << 60)), (LARGE, dict(n_dims=1 << 30)),
    (OK, dict(count=0)), (OK, dict(count=0, table=0)),
])
def test_rope_table(want, changed):
    assert status("tcrv_hip_rope_table", ROPE_TABLE, **changed) == want


ROPE = dict(elem=F32, layout=1, x=Q, x_token=4096, x_head=128, y=OUT, y_token=4096, y_head=128,
            positions=IDS, table=TABLE, table_rows=64, tokens=8, heads=32, head_dim=128, n_dims=64,
            inverse=0)


@pytest.mark.parametrize("want,changed", [
    (UNSUPPORTED, dict(elem=8)), (UNSUPPORTED, dict(elem=0)), (UNSUPPORTED, dict(layout=2)),
    (UNSUPPORTED, dict(layout=-1)), (SIZE, dict(n_dims=63)), (SIZE, dict(n_dims=130)),
    (SIZE, dict(x_head=127)), (SIZE, dict(y_head=64)), (SIZE, dict(x_token=127)),
    (SIZE, dict(y_token=0)), (NULL, dict(x=0)), (NULL, dict(y=0)), (NULL, dict(positions=0)),
    (NULL, dict(table=0)), (ALIGN, dict(x=Q + 2)), (ALIGN, dict(elem=F16, y=OUT + 1)),
    (ALIGN, dict(positions=IDS + 2)), (ALIGN, dict(table=TABLE + 1)),
    (LARGE, dict(tokens=1 << 31)), (LARGE, dict(heads=1 << 16)),
    (LARGE, dict(head_dim=65538, x_head=1 << 20, y_head=1 << 20, x_token=1 << 30,
                 y_token=1 << 30)),
    (OK, dict(tokens=0)), (OK, dict(heads=0)), (OK, dict(tokens=0, x=0, y=0, positions=0)),
])
def test_rope(want, changed):
    assert status("tcrv_hip_rope", ROPE, **changed) == want


TABLES = dict(context=IDS, added=IDS + 4096, requests=8, page_size=16, free=K, free_count=100,
              block_table=TABLE, stride=32, first=OUT, length=OUT + 4096, positions=V, slots=WS,
              max_tokens=64, taken=CACHE)


@pytest.mark.parametrize("want,changed", [
    (SIZE, dict(page_size=0)), (SIZE, dict(page_size=65537)), (NULL, dict(context=0)),
    (NULL, dict(added=0)), (NULL, dict(free=0)), (NULL, dict(block_table=0)), (NULL, dict(first=0)),
    (NULL, dict(length=0)), (NULL, dict(positions=0)), (NULL, dict(slots=0)), (NULL, dict(taken=0)),
    (ALIGN, dict(context=IDS + 2)), (ALIGN, dict(slots=WS + 4)), (ALIGN, dict(taken=CACHE + 1)),
    (ALIGN, dict(block_table=TABLE + 2)), (LARGE, dict(requests=1 << 31)),
    (LARGE, dict(max_tokens=1 << 31)), (LARGE, dict(stride=1 << 31)),
])
def test_tables(want, changed):
    assert status("tcrv_hip_kv_tables", TABLES, **changed) == want


STORE = dict(elem=F32, k=K, k_token=1024, k_head=128, v=V, v_token=1024, v_head=128, layout=1,
             positions=IDS, table=TABLE, table_rows=64, n_dims=128, slots=WS, cache=CACHE, pages=4,
             page_size=16, tokens=8, kv_heads=8, head_dim=128)
LOAD = dict(elem=F32, cache=CACHE, pages=4, page_size=16, slots=WS, k=K, k_token=1024, k_head=128,
            v=V, v_token=1024, v_head=128, tokens=8, kv_heads=8, head_dim=128)
ROWS = [
    (UNSUPPORTED, dict(elem=8)), (SIZE, dict(page_size=24)), (SIZE, dict(page_size=0)),
    (SIZE, dict(page_size=65552)), (SIZE, dict(head_dim=96)), (SIZE, dict(head_dim=32)),
    (SIZE, dict(head_dim=320)), (SIZE, dict(kv_heads=0)), (SIZE, dict(kv_heads=65536)),
    (SIZE, dict(k_head=100)), (SIZE, dict(v_token=64)), (NULL, dict(k=0)), (NULL, dict(v=0)),
    (NULL, dict(slots=0)), (NULL, dict(cache=0)), (ALIGN, dict(k=K + 2)),
    (ALIGN, dict(elem=BF16, v=V + 1)), (ALIGN, dict(slots=WS + 4)), (ALIGN, dict(cache=CACHE + 8)),
    (LARGE, dict(tokens=1 << 31)), (LARGE, dict(pages=1 << 31)), (OK, dict(tokens=0)),
]


@pytest.mark.parametrize("want,changed", ROWS + [
    (UNSUPPORTED, dict(layout=2)), (SIZE, dict(n_dims=129)), (SIZE, dict(n_dims=130)),
    (NULL, dict(positions=0)), (NULL, dict(table=0)), (ALIGN, dict(positions=IDS + 1)),
    (ALIGN, dict(table=TABLE + 2)), (OK, dict(tokens=0, n_dims=0, layout=7)),
])
def test_store(want, changed):
    assert status("tcrv_hip_kv_store_q4_0", STORE, **changed) == want


@pytest.mark.parametrize("want,changed", ROWS)
def test_load(want, changed):
    assert status("tcrv_hip_kv_load_q4_0", LOAD, **changed) == want


ATTN = dict(elem=F32, q=Q, q_token=4096, q_head=128, cache=CACHE, pages=64, page_size=16,
            block_table=TABLE, table_stride=8, first=IDS, length=IDS + 4096, requests=2, tokens=2,
            max_added=1, max_length=128, heads=32, kv_heads=8, head_dim=128, scale=0.1, causal=1,
            window=0, out=OUT, out_token=4096, out_head=128, workspace=WS, workspace_bytes=1 << 30)


@pytest.mark.parametrize("want,changed", [
    (UNSUPPORTED, dict(elem=8)), (SIZE, dict(heads=30)), (SIZE, dict(heads=0)),
    (SIZE, dict(kv_heads=0)), (SIZE, dict(head_dim=80)), (SIZE, dict(page_size=8)),
    (SIZE, dict(q_head=64)), (SIZE, dict(out_token=100)), (SIZE, dict(scale=float("nan"))),
    (SIZE, dict(scale=float("inf"))), (NULL, dict(q=0)), (NULL, dict(out=0)),
    (NULL, dict(cache=0)), (NULL, dict(block_table=0)), (NULL, dict(first=0)),
    (NULL, dict(length=0)), (ALIGN, dict(q=Q + 2)), (ALIGN, dict(elem=F16, out=OUT + 1)),
    (ALIGN, dict(cache=CACHE + 4)), (ALIGN, dict(block_table=TABLE + 2)),
    (ALIGN, dict(first=IDS + 1)), (ALIGN, dict(length=IDS + 2)), (LARGE, dict(requests=1 << 31)),
    (LARGE, dict(tokens=1 << 31)), (LARGE, dict(max_length=1 << 31)),
    (LARGE, dict(max_added=1 << 31)), (LARGE, dict(pages=1 << 31)),
    (LARGE, dict(table_stride=1 << 31)), (LARGE, dict(requests=1 << 20, max_added=1 << 20)),
    (OK, dict(tokens=0)), (OK, dict(requests=0)), (OK, dict(max_added=0)),
])
def test_attn(want, changed):
    assert status("tcrv_hip_attn_q4_0", ATTN, **changed) == want


def test_attn_workspace():
    """Long contexts of few requests need one; it is asked for and checked."""
    long = dict(max_length=65536, table_stride=4096)
    need = tcrv_hip.attn_q4_0_workspace_bytes("f32", 2, 2, 1, 65536, 32, 8, 128)
    assert need > 0
    assert status("tcrv_hip_attn_q4_0", ATTN, **long, workspace=0) == NULL
    assert status("tcrv_hip_attn_q4_0", ATTN, **long, workspace=WS + 4) == ALIGN
    assert status("tcrv_hip_attn_q4_0", ATTN, **long, workspace_bytes=need - 1) == SIZE
    for sizes in ((0, 2, 1, 65536, 32, 8, 128), (2, 0, 1, 65536, 32, 8, 128),
                  (2, 2, 1, 65536, 30, 8, 128), (2, 2, 1, 65536, 32, 8, 80),
                  (2, 2, 1, 1 << 40, 32, 8, 128)):
        assert tcrv_hip.attn_q4_0_workspace_bytes("f32", *sizes) == 0


@pytest.mark.parametrize("page,heads,dim,want", [
    (16, 1, 64, 16 * 72), (64, 8, 128, 64 * 8 * 144), (48, 2, 192, 48 * 2 * 216),
    (16, 3, 256, 16 * 3 * 288), (8, 1, 64, 0), (16, 0, 64, 0), (16, 1, 96, 0), (0, 1, 64, 0),
])
def test_page_bytes(page, heads, dim, want):
    """9/8 byte an element: two 4-bit quants, and two scales of two bytes for every 32."""
    assert tcrv_hip.kv_q4_0_page_bytes(page, heads, dim) == want


def test_floats_reach_the_library():
    """The double and float arguments' types: a wrong one would be read from another register."""
    assert tcrv_hip.SIGNATURES["tcrv_hip_attn_q4_0"][18] is ctypes.c_float
    assert tcrv_hip.SIGNATURES["tcrv_hip_rope_table"][2:8] == [ctypes.c_double] * 6
