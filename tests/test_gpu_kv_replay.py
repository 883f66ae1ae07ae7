"""A serving step captured once in a graph and replayed: what has to be moved on between replays is
the requests' contexts and the list of free pages."""
import numpy as np
import pytest
import torch

import kv_plain
from gpu_util import from_dev, to_dev

PAGE, WIDTH, PAGES = 16, 6, 12
CONTEXT = [10, 30]
HELD = [[5], [2, 9]]
FREE = [11, 3, 7, 0, 8, 1, 4, 6, 10]
STEPS = 37  # two pages more for the first request and three for the second, in different steps


def empty_table():
    table = np.full((2, WIDTH), -1, np.int32)
    for r, pages in enumerate(HELD):
        table[r, :len(pages)] = pages
    return table


def plain_steps(move):
    """The plain form's table after each step, with the list moved on by what was taken or left."""
    table, context, free, made = empty_table(), np.array(CONTEXT), list(FREE), []
    for _ in range(STEPS):
        got = kv_plain.tables(context, [1, 1], PAGE, np.array(free, np.int32), table, 2)
        table, context = got["block_table"], got["length"]
        if move:
            free = free[int(got["taken"][0]):] + [-1] * int(got["taken"][0])
        made.append(got)
    return made


def shared_pages(table):
    pages = table[table >= 0]
    return len(pages) - len(set(pages.tolist()))


def test_a_list_that_is_left_gives_pages_twice():
    assert shared_pages(plain_steps(move=False)[-1]["block_table"]) > 0
    last = plain_steps(move=True)[-1]["block_table"]
    assert shared_pages(last) == 0 and (last >= 0).sum() == 8


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["host", "graph"])
def test_replayed_steps(hip, dev, where):
    """The list moved on by the host's own count of pages, between replays, and on the device at the
    captured step's end.  Tables and slots as the plain form's, the cache's rows as they were stored,
    attention against float64 (an output is off by 2^-20 of the largest value and by 2^-20 |q||k| / 8
    of it, as in test_gpu_kv_cache.Setup)."""
    heads, dim, n = 2, 64, 2
    rng = np.random.default_rng(31)
    k, v = (rng.standard_normal((STEPS + 30, n, 1, dim)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((STEPS, n, heads, dim)).astype(np.float32)
    ints = lambda x, dtype=np.int32: to_dev(np.array(x, dtype), dev)  # noqa: E731
    context, added, free, table = ints(CONTEXT), ints([1, 1]), ints(FREE), to_dev(empty_table(), dev)
    first, length, positions, taken = ints([0] * 3), ints([0] * 2), ints([0] * 2), ints([0])
    slots = ints([0] * 2, np.int64)
    cache = torch.full((PAGES * hip.kv_q4_0_page_bytes(PAGE, 1, dim),), 0xFF, dtype=torch.uint8, device=dev)
    dk, dv = (torch.zeros(n, 1, dim, device=dev) for _ in range(2))
    dq, out = (torch.zeros(n, heads, dim, device=dev) for _ in range(2))
    bounds = 1, WIDTH * PAGE
    need = hip.attn_q4_0_workspace_bytes("f32", n, n, *bounds, heads, 1, dim)
    ws = torch.zeros(max(need, 16), dtype=torch.uint8, device=dev)
    for r, c in enumerate(CONTEXT):  # the tokens of before
        at = ints([HELD[r][t // PAGE] * PAGE + t % PAGE for t in range(c)], np.int64)
        old = [to_dev(x[:c, r], dev) for x in (k, v)]
        hip.kv_store_q4_0("f32", old[0], dim, dim, old[1], dim, dim, "half", None, None, 0, 0, at, cache,
                          PAGES, PAGE, c, 1, dim)
    place = torch.arange(len(FREE), device=dev)

    def step():
        hip.kv_tables(context, added, n, PAGE, free, len(FREE), table, WIDTH, first, length, positions,
                      slots, n, taken)
        hip.kv_store_q4_0("f32", dk, dim, dim, dv, dim, dim, "half", None, None, 0, 0, slots, cache,
                          PAGES, PAGE, n, 1, dim)
        hip.attn_q4_0("f32", dq, heads * dim, dim, cache, PAGES, PAGE, table, WIDTH, first, length, n, n,
                      *bounds, heads, 1, dim, dim ** -0.5, True, 0, out, heads * dim, dim, ws, need)
        if where == "graph":
            after = place + taken
            moved = torch.where(after < len(FREE), free[after.clamp(max=len(FREE) - 1)], -1)
            free.copy_(moved)
            context.copy_(length)

    # Once before the capture, on the side and on copies of what it changes
    kept = [x.clone() for x in (context, free, table, cache)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    for x, y in zip((context, free, table, cache), kept):
        x.copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    torch.cuda.synchronize()

    left, before = list(FREE), list(CONTEXT)
    for i, want in enumerate(plain_steps(move=True)):
        for buf, x in ((dk, k), (dv, v)):
            buf.copy_(to_dev(np.stack([x[before[r], r] for r in range(n)]), dev))
        dq.copy_(to_dev(q[i], dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(from_dev(table), want["block_table"]), i
        assert np.array_equal(from_dev(slots), want["slots"]) and shared_pages(from_dev(table)) == 0
        new = sum(-(-(c + 1) // PAGE) - -(-c // PAGE) for c in before)
        assert new == int(from_dev(taken)[0])
        before = [c + 1 for c in before]
        if where == "host":
            left = left[new:]
            free.copy_(ints(left + [-1] * (len(FREE) - len(left))))
            context.copy_(ints(before))
        else:
            assert np.array_equal(from_dev(context), before)
        got = from_dev(out)
        for r, c in enumerate(before):
            keys, vals = (kv_plain.values(*kv_plain.quantize(x[:c, r])) for x in (k, v))
            ref = kv_plain.attend(q[i][r:r + 1], keys, vals, c - 1, dim ** -0.5, True, 0)
            qk = np.linalg.norm(q[i][r], axis=-1).max() * np.linalg.norm(keys, axis=-1).max() / 8
            tol = 2 * np.abs(vals).max() * (2.0 ** -21 * qk + 2.0 ** -20)
            assert np.abs(got[r] - ref[0]).max() <= tol, (i, r)
