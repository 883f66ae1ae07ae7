"""Strides of the rows that the cache's entries write: layouts whose rows would share places are
refused before any launch, all others launch (tests/launches.py), on the CPU."""
import itertools
import random

import pytest

import launches
import tcrv_hip
from tcrv_hip import ERR_BAD_SIZE, OK

A, B, C, D, E, F, G = ((i + 1) << 40 for i in range(7))


def rope(tokens, heads, dim, token, head, same=False):
    x = (token, head) if same else (heads * dim, dim)
    return "tcrv_hip_rope", (7, 1, A, *x, A if same else B, token, head, C, D, 64, tokens, heads,
                             dim, 0, 0)


def load(tokens, heads, dim, token, head, which="k"):
    k, v = (heads * dim, dim), (token, head)
    k, v = (v, k) if which == "k" else (k, v)
    return "tcrv_hip_kv_load_q4_0", (7, A, 64, 16, B, C, *k, D, *v, tokens, heads, dim)


def attn(tokens, heads, dim, token, head):
    return "tcrv_hip_attn_q4_0", (7, A, heads * dim, dim, B, 64, 16, C, 8, D, E, tokens, tokens, 1, 64,
                                  heads, heads, dim, 0.1, 1, 0, F, token, head, G, 1 << 40)


ENTRIES = [rope, lambda *a: rope(*a, same=True), load, lambda *a: load(*a, which="v"), attn]


@pytest.mark.parametrize("entry", range(len(ENTRIES)))
@pytest.mark.parametrize("tokens,heads,token,head,want", [
    (3, 2, 128, 64, OK), (3, 2, 127, 64, ERR_BAD_SIZE),   # token by token
    (3, 2, 64, 192, OK), (3, 2, 64, 191, ERR_BAD_SIZE),   # head by head
    (2, 2, 192, 128, OK), (3, 2, 96, 64, ERR_BAD_SIZE), (9, 3, 96, 64, ERR_BAD_SIZE),
    (3, 2, 64, 64, ERR_BAD_SIZE), (2, 2, 64, 64, ERR_BAD_SIZE), (1, 2, 64, 64, OK), (2, 1, 64, 64, OK),
    (100, 2, 128, 192, OK), (100, 2, 128, 190, ERR_BAD_SIZE),  # heads in the tokens' gaps
    (100, 3, 128, 192, ERR_BAD_SIZE), (2, 3, 64, 128, OK),
    (1 << 20, 2, 1 << 62, (1 << 62) + 64, OK), (1 << 20, 2, 1 << 62, 1 << 62, ERR_BAD_SIZE),
])
def test_rows_that_are_written(entry, tokens, heads, token, head, want):
    call = ENTRIES[entry](tokens, heads, 64, token, head)
    (status, made), = launches.replay([call])
    assert status == want and bool(made) == (want == OK)


def test_all_small_layouts():
    """Against the places themselves."""
    rng = random.Random(5)
    calls, want = [], []
    for _ in range(400):
        tokens, heads, dim = rng.randint(1, 6), rng.randint(1, 6), rng.choice((1, 2, 5))
        token, head = rng.randint(1, 40), rng.randint(1, 40)
        places = [t * token + h * head + i for t, h, i in itertools.product(range(tokens), range(heads),
                                                                            range(dim))]
        calls.append(rope(tokens, heads, dim, token, head))
        want.append(OK if len(set(places)) == len(places) else ERR_BAD_SIZE)
    got = [status for status, _ in launches.replay(calls)]
    # a stride of less than a row is refused where rows follow one another by it, as before
    assert got == want
    assert 80 < sum(s == OK for s in got) < 320


def test_rows_that_are_read_may_overlap():
    q = ("tcrv_hip_rope", (7, 1, A, 96, 64, B, 128, 64, C, D, 64, 3, 2, 64, 0, 0))
    k = ("tcrv_hip_kv_store_q4_0", (7, A, 96, 64, B, 96, 64, 1, 0, 0, 0, 0, C, D, 64, 16, 3, 2, 64))
    assert [status for status, _ in launches.replay([q, k])] == [OK, OK]
