"""Which kernels attn_q4_0 launches at a size and the grids they get, replayed without a GPU
(tests/launches.py); and that the workspace query covers every window."""
import re

import pytest

import launches
import tcrv_hip


def attn(elem, requests, tokens, most_added, most_length, heads, kv, dim, window=0, causal=1,
         ws=1 << 50, pages=1 << 20):
    q, out, cache, ints, work = ((k + 1) << 40 for k in range(5))
    return "tcrv_hip_attn_q4_0", (
        tcrv_hip.FLOAT_ELEM[elem], q, heads * dim, dim, cache, pages, 16, ints, 1 << 16, ints + (1 << 30),
        ints + (2 << 30), requests, tokens, most_added, most_length, heads, kv, dim, dim ** -0.5, causal,
        window, out, heads * dim, dim, work, ws)


def run(*args, **kw):
    status, made = launches.replay([attn(*args, **kw)])[0]
    assert status == 0
    # names of f16 instances come mangled
    return [(re.search("attn_q4_0_(rows16|tiles|join_few|join)", x.name)[1], x.grid) for x in made]


@pytest.mark.parametrize("args,want", [
    # decode: short contexts on a work-group a tile, longer ones shared out and joined
    (("f16", 64, 64, 1, 512, 32, 8, 128), [("rows16", 512)]),
    (("f16", 64, 64, 1, 2560, 32, 8, 128), [("rows16", 512)]),
    (("f16", 64, 64, 1, 2561, 32, 8, 128), [("rows16", 512), ("join_few", 512)]),
    (("f16", 64, 64, 1, 8192, 32, 8, 256), [("rows16", 256), ("join_few", 256)]),
    (("f32", 1, 1, 1, 300, 32, 8, 128), [("rows16", 16), ("join_few", 16)]),
    (("f32", 1, 1, 1, 33, 32, 8, 128), [("rows16", 8)]),
    # drafted tokens: up to 64 rows where there are work-groups enough
    (("f16", 8, 128, 16, 1000, 32, 8, 128), [("rows16", 256)]),
    (("f16", 4, 64, 16, 100, 32, 8, 128), [("tiles", 32)]),
    # prompts: whole tiles where they are many, parts of them where they are few
    (("f16", 1, 4096, 4096, 4096, 32, 8, 128), [("tiles", 512)]),
    (("f16", 1, 64, 64, 16384, 32, 8, 128), [("tiles", 512), ("join", 64)]),
    # both kinds
    (("f32", 9, 600, 300, 300, 14, 2, 64), [("rows16", 36), ("join_few", 36), ("tiles", None), ("join", 600)]),
])
def test_kernels_of_a_size(args, want):
    got = run(*args)
    assert [n for n, _ in got] == [n for n, _ in want], got
    for (_, grid), (_, groups) in zip(got, want):
        if groups is not None:
            assert grid[0] == groups, got


@pytest.mark.parametrize("elem", ["f32", "f16", "bf16"])
def test_nothing_to_do_launches_nothing(elem):
    for args in ((elem, 0, 5, 1, 9, 4, 2, 64), (elem, 3, 0, 1, 9, 4, 2, 64), (elem, 3, 5, 0, 9, 4, 2, 64)):
        assert run(*args) == []


@pytest.mark.parametrize("requests,tokens,added,heads,kv,dim", [
    (1, 1, 1, 32, 8, 128), (64, 64, 1, 32, 8, 128), (5, 700, 300, 14, 2, 64), (3, 90, 30, 16, 4, 256),
    (200, 200, 1, 10, 2, 192), (1, 2000, 2000, 8, 8, 128),
])
@pytest.mark.parametrize("length", [1, 257, 4000, 131072, 1 << 30])
def test_workspace_serves_every_window(requests, tokens, added, heads, kv, dim, length):
    calls, need = [], tcrv_hip.attn_q4_0_workspace_bytes("f16", requests, tokens, added, length, heads,
                                                         kv, dim)
    for window in (0, 1, 100, 1000, 5000, 1 << 40):
        for causal in (0, 1):
            calls.append(attn("f16", requests, tokens, added, length, heads, kv, dim, window, causal,
                              ws=need))
    assert all(status == 0 for status, _ in launches.replay(calls))
    if need:  # and no less does without a window
        status, made = launches.replay([attn("f16", requests, tokens, added, length, heads, kv, dim,
                                             ws=need - 1)])[0]
        assert status == tcrv_hip.ERR_BAD_SIZE and not made
