"""Calls of the cache's entries near the most that a launch holds, 2^32 - 1 threads along an axis, on the
CPU (tests/launches.py): what launches lies within it, and what does not fit is refused before
anything is launched."""
import pytest

import launches
from tcrv_hip import ERR_TOO_LARGE, OK

A, B, C, D, E, F, G = ((i + 1) << 50 for i in range(7))


def rope(tokens):
    return "tcrv_hip_rope", (9, 1, A, 2, 2, B, 2, 2, C, D, 64, tokens, 1, 2, 2, 0)


def table(count):
    return "tcrv_hip_rope_table", (0, 2, 1e4, 1.0, 1.0, 1.0, 1.0, 0.0, 0, 0, count, A)


def store(tokens):
    return "tcrv_hip_kv_store_q4_0", (9, A, 64, 64, B, 64, 64, 1, 0, 0, 0, 0, C, D, 64, 16, tokens, 1,
                                      64)


def load(tokens):
    return "tcrv_hip_kv_load_q4_0", (9, A, 64, 16, B, C, 64, 64, D, 64, 64, tokens, 1, 64)


def attn(requests, tokens, added, length=16, heads=1, kv=1, dim=64):
    return "tcrv_hip_attn_q4_0", (9, A, heads * dim, dim, B, 64, 16, C, 8, D, E, requests, tokens, added,
                                  length, heads, kv, dim, 0.1, 1, 0, F, heads * dim, dim, G, 1 << 60)


MOST = (1 << 24) - 1


@pytest.mark.parametrize("call,want", [
    (rope(MOST), OK), (rope(MOST + 1), ERR_TOO_LARGE),
    (table(16 * MOST), OK), (table(16 * MOST + 1), ERR_TOO_LARGE),
    (store(MOST), OK), (store(MOST + 1), ERR_TOO_LARGE),
    (load(MOST), OK), (load(MOST + 1), ERR_TOO_LARGE),
    (attn(MOST, MOST, 1), OK), (attn(MOST + 1, MOST + 1, 1), ERR_TOO_LARGE),
    # a work-group a tile: short contexts of many requests
    (attn(1 << 20, 1 << 20, 1, heads=15, kv=15), OK),
    (attn(1 << 20, 1 << 20, 1, heads=16, kv=16), ERR_TOO_LARGE),
    # prompts, of 512 threads a tile, and of 256
    (attn(1, MOST, MOST, heads=127, kv=127), OK),
    (attn(1, MOST, MOST, heads=128, kv=128), ERR_TOO_LARGE),
    (attn(1, MOST, MOST, heads=127, kv=127, dim=256), OK),
    (attn(1, MOST, MOST, heads=128, kv=128, dim=256), ERR_TOO_LARGE),
    # both kernels: neither is launched where one does not fit
    (attn(1 << 18, 1 << 19, 128, heads=70, kv=70), ERR_TOO_LARGE),
    # few rows, and room for more tokens than they have
    (attn(1, MOST + 1, 64, 4096, heads=4), ERR_TOO_LARGE),
])
def test_most_that_a_launch_holds(call, want):
    (status, made), = launches.replay([call])
    assert status == want
    assert bool(made) == (want == OK)
    for x in made:
        assert all(g * b < 1 << 32 for g, b in zip(x.grid, x.block)), made
