"""Values that are not finite among the keys that only some of a sequence's rows see, in the kernel that takes few rows:
clusters, whole items and shared lines, up to 8 rows and up to 16, with and without a prefix, several items a CTA."""
import math

import pytest
import torch

from attn_ref import check
from nebula_b200 import hq
from test_gpu_attn import BF16, F16, gen, paged_case, paged_ref, run_paged

pytestmark = pytest.mark.gpu


def place(c, s, key, head, dim, value):
    """A value of sequence s's key, in the pages and in the reference's copy."""
    page_size = c["v"].shape[1]
    c["v"][c["table"][s, key // page_size].long(), key % page_size, head, dim] = value
    c["keys"][s][1][key, head, dim] = value


CASES = [
    # heads, kv heads, head dim, type, lengths, rows, page, prefix, layout
    # few items: a cluster each, up to 8 rows and up to 16, keys that end inside a unit and at its end
    (5, 1, 128, F16, [300], [3], 16, 0, "nhd"),
    (4, 4, 128, BF16, [700, 256], [8, 5], 32, 0, "nhd"),
    (10, 2, 64, BF16, [1000, 130], [3, 2], 16, 100, "hnd"),
    (16, 1, 64, F16, [90], [1], 16, 0, "nhd"),
    (2, 2, 96, F16, [500], [16], 16, 40, "nhd"),
    (1, 1, 40, BF16, [129], [15], 16, 0, "nhd"),
    # as many keys as rows, and fewer
    (2, 1, 128, F16, [5, 3], [5, 6], 16, 0, "nhd"),
    # many short items: a CTA takes several
    (10, 2, 128, F16, [20 + 3 * i % 90 for i in range(300)], [3] * 300, 16, 0, "nhd"),
    (8, 8, 64, BF16, [16 + i % 50 for i in range(80)], [4] * 80, 16, 30, "nhd"),
    (8, 4, 128, BF16, [40 + 7 * i % 200 for i in range(120)], [8 - i % 3 for i in range(120)], 32, 0, "hnd"),
    # lines that CTAs share
    (4, 2, 128, BF16, [20000, 3, 15000, 9000], [2, 1, 2, 2], 64, 0, "nhd"),
    (6, 2, 64, F16, [(41 * i) % 2000 + 4 for i in range(300)], [4] * 300, 16, 0, "nhd"),
    (6, 2, 64, F16, [(41 * i) % 2000 + 4 for i in range(300)], [5] * 300, 16, 129, "nhd"),
    # beside the kernel of many rows
    (5, 1, 128, F16, [200, 900, 60, 300], [1, 60, 1, 1], 16, 0, "nhd"),
    (4, 4, 64, BF16, [200, 900, 60, 300], [4, 60, 8, 2], 16, 0, "nhd"),
]


@pytest.mark.parametrize("Hq,Hk,D,dt,lens,rows,page,prefix,layout", CASES)
def test_values_of_a_sequences_last_keys(Hq, Hk, D, dt, lens, rows, page, prefix, layout):
    """NaN, +Inf and -Inf, also two of them in one dim, in every second sequence: they reach the rows that see their
    key, and nothing else -- neither the rows before it nor the items around it."""
    c = paged_case(Hq, Hk, D, dt, lens, rows, page, prefix, layout, seed=len(lens) + sum(rows))
    values = (math.nan, math.inf, -math.inf)
    for s in range(0, len(lens), 2):
        n = min(rows[s], lens[s])
        for i in range(n):  # each of the last n keys, the first of them seen by all rows
            key, h = lens[s] - n + i, (s + i) % Hk
            place(c, s, key, h, (11 * s + 5 * i) % D, values[(s // 2 + i) % 3])
            if i % 2:
                place(c, s, key, h, (11 * s + 5 * (i - 1)) % D, values[(s // 2 + i + 1) % 3])
    o, _, m = paged_ref(c)
    n = c["cu_host"][-1]
    assert not bool(torch.isfinite(o).all())
    for _ in range(3):
        check(run_paged(c)[:n], o, m, dt)
    hq.check_device_error()


def test_the_next_item_of_a_cta_begins_clean():
    """What one item's rows had put back does not stay for the next one: only the first sequences hold such values."""
    B, n = 300, 3
    c = paged_case(10, 2, 128, BF16, [100 + i % 64 for i in range(B)], [n] * B, 16, 0, seed=2)
    for s in range(B // 2):
        for i in range(n):
            place(c, s, int(c["lens"][s]) - n + i, i % 2, 7 * i, math.inf if i % 2 else math.nan)
    o, _, m = paged_ref(c)
    got = run_paged(c)[: B * n]
    assert bool(torch.isfinite(got[B // 2 * n:]).all())
    check(got, o, m, BF16)
    hq.check_device_error()


def test_captured_steps_with_values_that_come_and_go():
    """A replayed call over the same pages, with and without such values."""
    c = paged_case(5, 1, 128, F16, [3000, 400, 77, 15], [3] * 4, 16, 0, seed=3, poison=False)
    out = torch.zeros_like(c["q"])
    run_paged(c, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_paged(c, out=out)
    n = c["cu_host"][-1]
    for value in (math.nan, 1.5, -math.inf, 0.25):
        for s in range(4):
            place(c, s, int(c["lens"][s]) - 1 - s % 3, 0, 100, value)
        c["q"].copy_(torch.randn(c["q"].shape, generator=gen(4), device="cuda", dtype=F16))
        graph.replay()
        o, _, m = paged_ref(c)
        check(out[:n], o, m, F16)
    hq.check_device_error()
