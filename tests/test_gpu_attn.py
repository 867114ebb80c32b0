"""Attention kernels against the definition in 64 bits, at the sizes, layouts and masks where they can go wrong."""
import math

import pytest
import torch

from attn_ref import attend, check, check_lse
from nebula_b200 import _lib, hq
from nebula_b200 import attention as at

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def qkv_rows(T, Hq, Hk, D, dt, g):
    """q, k, v as slices of one buffer, as the QKV layer writes them."""
    x = torch.randn((T, (Hq + 2 * Hk) * D), generator=g, device="cuda", dtype=dt)
    a, b = Hq * D, (Hq + Hk) * D
    return x[:, :a].view(T, Hq, D), x[:, a:b].view(T, Hk, D), x[:, b:].view(T, Hk, D)


def prompt_ref(q, k, v, cu, scale, causal=True):
    outs, lses, mags = [], [], []
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        seen = torch.arange(1, n + 1) if causal else torch.full((n,), n)
        o, l, m = attend(q[a:b], k[a:b], v[a:b], seen, scale)
        outs.append(o), lses.append(l), mags.append(m)
    return torch.cat(outs), torch.cat(lses), torch.cat(mags)


PROMPTS = [
    # heads, kv heads, head dim, type, lengths, causal
    (1, 1, 8, F16, [1], True),
    (4, 2, 64, BF16, [1, 2, 3], True),
    (5, 1, 128, F16, [0, 25, 0, 26, 1], True),
    (10, 2, 128, BF16, [51, 52, 103, 7], True),
    (40, 8, 128, BF16, [257], True),
    (16, 16, 64, F16, [127, 128, 129, 1], True),
    (16, 16, 64, F16, [255, 256, 257], False),
    (3, 3, 40, F16, [300], True),
    (6, 2, 96, BF16, [129, 500], True),
    (24, 1, 72, F16, [33, 64], True),
    (8, 8, 120, BF16, [640], False),
    (32, 4, 128, F16, [1100], True),
    (5, 1, 128, BF16, [2500, 1, 37], True),
    # more blocks than SMs, of very different lengths
    (16, 16, 64, F16, [700, 90, 1, 512, 333, 0, 256, 601, 44, 129, 700, 511], True),
    (40, 8, 128, BF16, [600, 128, 601, 37, 400], True),
    (20, 20, 128, F16, [1024, 300], False),
    # as many query heads a key/value head as a tile has rows, and numbers that leave rows of it idle
    (128, 1, 64, BF16, [5, 40], True),
    (100, 1, 128, F16, [3, 130], True),
    (86, 2, 8, F16, [70], True),
    (21, 3, 64, BF16, [19, 150], False),
]


@pytest.mark.parametrize("Hq,Hk,D,dt,lens,causal", PROMPTS)
def test_prompt(Hq, Hk, D, dt, lens, causal):
    T = sum(lens) + 3  # three rows behind the last sequence
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    q, k, v = qkv_rows(T, Hq, Hk, D, dt, gen(T * Hq + D))
    q[cu[-1]:], k[cu[-1]:], v[cu[-1]:] = math.nan, math.nan, math.inf
    out = torch.full((T, Hq, D), 7.0, dtype=dt, device="cuda")
    lse = torch.full((T, Hq), 7.0, device="cuda")
    got = at.attn_prompt(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), max(lens), causal=causal, out=out,
                         lse=lse)
    assert got is out
    o, l, m = prompt_ref(q, k, v, cu, D ** -0.5, causal)
    n = cu[-1]
    check(got[:n], o, m, dt)
    check_lse(lse[:n], l)
    assert bool((got[n:] == 7).all()) and bool((lse[n:] == 7).all())
    hq.check_device_error()


def test_prompt_scale_and_repeat():
    """Another scale, sharp softmax; the same call twice gives the same bits."""
    q, k, v = qkv_rows(700, 8, 2, 128, F16, gen(1))
    cu = torch.tensor([0, 333, 700], dtype=torch.int32, device="cuda")
    a = at.attn_prompt(q, k, v, cu, 367, scale=0.5)
    b = at.attn_prompt(q, k, v, cu, 367, scale=0.5)
    assert torch.equal(a, b)
    o, _, m = prompt_ref(q, k, v, [0, 333, 700], 0.5)
    # scores of up to sum |q k| / 2 ~ 41: 128 x 2^-24 x 41
    check(a, o, m, F16, score_error=4e-4)


@pytest.mark.parametrize("D,dt", [(128, BF16), (64, F16)])
@pytest.mark.parametrize("where", [0, 5, 130, 299])
def test_prompt_values_that_are_not_finite(D, dt, where):
    """What a later token holds does not reach earlier rows; what a row sees does."""
    q, k, v = qkv_rows(300, 4, 2, D, dt, gen(where))
    v[where, 0, 3] = math.nan
    v[where, 1, 7] = math.inf
    v[where, 1, 8] = -math.inf
    got = at.attn_prompt(q, k, v, torch.tensor([0, 300], dtype=torch.int32, device="cuda"), 300)
    o, _, m = prompt_ref(q, k, v, [0, 300], D ** -0.5)
    check(got, o, m, dt)


@pytest.mark.parametrize("where", [0, 77, 299])
def test_prompt_keys_that_are_not_finite(where):
    q, k, v = qkv_rows(300, 4, 2, 128, BF16, gen(where))
    k[where, 1, 3] = math.nan
    got = at.attn_prompt(q, k, v, torch.tensor([0, 300], dtype=torch.int32, device="cuda"), 300)
    o, _, m = prompt_ref(q, k, v, [0, 300], 128 ** -0.5)
    assert bool(torch.isnan(got[where:, 2:]).all()) and not bool(torch.isnan(got[:where]).any())
    check(got, o, m, BF16)


def test_prompt_growing_scores():
    """Scores that grow along the keys: the running maximum moves at every tile, by little and by much."""
    for step in (0.02, 1.0, 30.0):
        T, D = 600, 64
        g = gen(3)
        q = torch.ones((T, 2, D), device="cuda", dtype=BF16)
        k = (torch.arange(T, device="cuda", dtype=torch.float32) * step / D)[:, None, None].expand(T, 1, D).to(BF16)
        v = torch.randn((T, 1, D), generator=g, device="cuda", dtype=BF16)
        got = at.attn_prompt(q, k.contiguous(), v, torch.tensor([0, T], dtype=torch.int32, device="cuda"), T, scale=1.0)
        o, _, m = prompt_ref(q, k.contiguous(), v, [0, T], 1.0)
        # sum |q k| = up to 600 step: 128 x 2^-24 of it, and 2^-23 of the exponent's argument
        check(got, o, m, BF16, score_error=1e-4 + 600 * step * 130 * 2.0 ** -24)


def paged_case(Hq, Hk, D, dt, lens, q_lens, page, prefix, layout="nhd", seed=0, poison=True):
    g = gen(seed)
    used = [-(-n // page) for n in lens]
    pre = -(-prefix // page)
    num = sum(used) + pre + 2
    shape = {"nhd": (num, page, Hk, D), "hnd": (num, Hk, page, D), "kv": (num, 2, page, Hk, D)}[layout]
    if layout == "kv":
        both = torch.randn(shape, generator=g, device="cuda", dtype=dt)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (torch.randn(shape, generator=g, device="cuda", dtype=dt) for _ in range(2))
        if layout == "hnd":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
    perm = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(used + [1])), -7, dtype=torch.int32, device="cuda")
    i = 0
    keep = torch.zeros((num, page), dtype=torch.bool, device="cuda")
    keys = []
    for s, n in enumerate(lens):
        mine = perm[i: i + used[s]]
        table[s, : used[s]] = mine
        i += used[s]
        at_ = torch.arange(n, device="cuda")
        where = (mine[at_ // page].long(), at_ % page)
        keep[where] = True
        keys.append((k[where], v[where]))
    ptab = perm[i: i + pre].clone()
    at_ = torch.arange(prefix, device="cuda")
    where = (ptab[at_ // page].long(), at_ % page) if prefix else None
    pkv = (k[where], v[where]) if prefix else (k[:0, 0], v[:0, 0])
    if prefix:
        keep[where] = True
    if poison:  # stale slots hold anything
        k[~keep], v[~keep] = math.nan, math.inf
    T = sum(q_lens) + 2
    q = torch.randn((T, Hq, D), generator=g, device="cuda", dtype=dt)
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    return dict(q=q, k=k, v=v, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q=max(q_lens + [0]), ptab=ptab, prefix=prefix,
                cu_host=cu, keys=keys, pkv=pkv, dt=dt, scale=D ** -0.5)


def paged_ref(c):
    outs, lses, mags = [], [], []
    for s, (k, v) in enumerate(c["keys"]):
        a, b = c["cu_host"][s], c["cu_host"][s + 1]
        n, m = b - a, k.shape[0]
        seen = c["prefix"] + (m - n + 1 + torch.arange(n)).clamp(min=0)
        o, l, g = attend(c["q"][a:b], torch.cat([c["pkv"][0], k]), torch.cat([c["pkv"][1], v]), seen, c["scale"])
        outs.append(o), lses.append(l), mags.append(g)
    return torch.cat(outs), torch.cat(lses), torch.cat(mags)


def run_paged(c, **kw):
    kw = dict(dict(prefix_table=c["ptab"] if c["prefix"] else None, prefix_len=c["prefix"]), **kw)
    return at.attn_paged(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], c["max_q"], **kw)


PAGED = [
    # heads, kv heads, head dim, type, lengths, rows, page, prefix, layout
    (1, 1, 8, F16, [1], [1], 16, 0, "nhd"),
    (40, 8, 128, BF16, [777], [1], 16, 0, "nhd"),
    (40, 8, 128, F16, [1, 15, 16, 17, 127, 128, 129, 1000], [1] * 8, 16, 0, "hnd"),
    (10, 2, 128, BF16, [0, 5, 0, 300, 31], [1] * 5, 32, 0, "kv"),
    (5, 1, 128, F16, [5000, 1, 64], [1] * 3, 64, 0, "nhd"),
    (16, 16, 64, BF16, [33, 700, 256], [1] * 3, 128, 0, "hnd"),
    (16, 1, 64, F16, [90, 2000], [1, 1], 16, 0, "nhd"),
    (17, 1, 64, F16, [90, 2000], [1, 1], 16, 0, "nhd"),
    (64, 1, 128, BF16, [90, 2000], [1, 1], 256, 0, "nhd"),
    (3, 3, 40, F16, [50, 300], [1, 1], 16, 0, "nhd"),
    (6, 3, 96, BF16, [50, 300], [2, 1], 16, 0, "hnd"),
    (10, 2, 128, F16, [3, 60], [3, 3], 16, 0, "nhd"),
    # more rows than keys: the first rows see nothing
    (10, 2, 128, F16, [2, 0], [3, 2], 16, 0, "nhd"),
    (5, 1, 128, BF16, [10, 300, 500, 70], [1, 64, 1, 70], 16, 0, "nhd"),
    (40, 8, 128, F16, [900, 31, 1500], [1, 1, 64], 16, 0, "nhd"),
    (8, 8, 64, BF16, [4000], [130], 64, 0, "hnd"),
    (32, 4, 128, F16, [40, 1111], [40, 1111], 32, 0, "nhd"),
    # no rows for a sequence that has keys
    (10, 2, 128, BF16, [40, 50], [0, 1], 16, 0, "nhd"),
    # shared prefixes: shorter than a page, whole pages, long; sequences without own keys
    (5, 1, 128, F16, [20, 3], [1, 1], 16, 7, "nhd"),
    (10, 2, 128, BF16, [20, 3, 150], [1] * 3, 16, 1024, "nhd"),
    (40, 8, 128, BF16, [100, 0, 1, 260], [1] * 4, 64, 3001, "hnd"),
    (16, 16, 64, F16, [5, 6, 7], [1] * 3, 32, 129, "nhd"),
    (8, 1, 64, BF16, [80, 9], [70, 9], 16, 200, "nhd"),
    (40, 8, 128, F16, [12] * 60, [1] * 60, 16, 515, "nhd"),
    (24, 2, 80, F16, [40, 41], [1, 30], 16, 333, "kv"),
    # many short streams: groups of 4, 2 and 1 warps an item, in one round and in several
    (40, 8, 128, BF16, [1 + 7 * i % 60 for i in range(25)], [1] * 25, 16, 0, "nhd"),
    (16, 8, 64, F16, [1 + 5 * i % 40 for i in range(64)], [1] * 64, 16, 0, "hnd"),
    (10, 10, 128, F16, [i % 33 for i in range(130)], [1] * 130, 16, 0, "nhd"),
    (8, 8, 64, BF16, [1 + i % 47 for i in range(333)], [1] * 333, 16, 0, "nhd"),
    (8, 8, 64, BF16, [1 + i % 47 for i in range(333)], [1] * 333, 16, 100, "nhd"),
    # lines of units that CTAs share: one long stream, several, more sequences than threads, empty ones between
    (2, 2, 128, F16, [20000], [1], 64, 0, "nhd"),
    (10, 2, 64, BF16, [0, 9000, 1, 0, 12000, 17, 0], [1] * 7, 128, 0, "hnd"),
    (3, 1, 64, F16, [(37 * i) % 2000 for i in range(300)], [1] * 300, 16, 0, "nhd"),
    (3, 1, 64, F16, [(37 * i) % 2000 for i in range(300)], [1] * 300, 16, 77, "nhd"),
    (10, 2, 128, BF16, [20000, 3, 15000], [1] * 3, 64, 500, "nhd"),
    (30, 2, 128, BF16, [20000, 3, 15000], [1] * 3, 64, 0, "nhd"),
    (4, 2, 64, F16, [20000, 3, 15000], [4, 2, 3], 64, 129, "nhd"),
    # chunks beside streams that CTAs share
    (10, 2, 128, F16, [3000, 9000, 40, 13500], [1, 1, 1, 100], 16, 0, "nhd"),
    (24, 2, 64, BF16, [3000, 9000, 40, 13500], [1, 100, 1, 1], 16, 300, "hnd"),
    (64, 1, 64, F16, [300, 900], [1, 2], 16, 40, "nhd"),
    (128, 1, 128, BF16, [300, 900], [1, 2], 16, 0, "nhd"),
    # a few rows each of many sequences
    (10, 2, 128, F16, [20 + 9 * i for i in range(100)], [4 - i % 4 for i in range(100)], 16, 0, "nhd"),
    (5, 1, 64, BF16, [20 + 9 * i for i in range(100)], [4] * 100, 32, 50, "nhd"),
    # a prefix under more rows than the SMs take at once
    (16, 16, 64, F16, [600, 601, 40], [600, 300, 1], 32, 200, "nhd"),
]


@pytest.mark.parametrize("Hq,Hk,D,dt,lens,rows,page,prefix,layout", PAGED)
def test_paged(Hq, Hk, D, dt, lens, rows, page, prefix, layout):
    c = paged_case(Hq, Hk, D, dt, lens, rows, page, prefix, layout, seed=len(lens) + sum(lens))
    T, n = c["q"].shape[0], c["cu_host"][-1]
    out = torch.full((T, Hq, D), 7.0, dtype=dt, device="cuda")
    lse = torch.full((T, Hq), 7.0, device="cuda")
    got = run_paged(c, out=out, lse=lse)
    o, l, m = paged_ref(c)
    check(got[:n], o, m, dt)
    check_lse(lse[:n], l)
    assert bool((got[n:] == 7).all()) and bool((lse[n:] == 7).all())
    assert torch.equal(run_paged(c)[:n], got[:n])  # and the same bits again
    hq.check_device_error()


@pytest.mark.parametrize("prefix", [0, 100])
def test_paged_one_row_each_without_offsets(prefix):
    c = paged_case(10, 2, 128, F16, [30, 500, 2], [1] * 3, 16, prefix, seed=4)
    want = run_paged(c)
    got = at.attn_paged(c["q"][:3], c["k"], c["v"], c["table"], c["lens"], max_kv_len=500,
                        prefix_table=c["ptab"] if prefix else None, prefix_len=prefix)
    assert torch.equal(got, want[:3])


def test_paged_bound_does_not_change_the_result():
    """max_kv_len sizes the launch only: too small or much too large, the rows are right."""
    c = paged_case(10, 2, 128, BF16, [30, 2500, 2], [1, 20, 1], 16, 0, seed=5)
    o, _, m = paged_ref(c)
    n = c["cu_host"][-1]
    for bound in (1, 2500, 1 << 20):
        check(run_paged(c, max_kv_len=bound)[:n], o, m, BF16)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_paged_strided_rows(dt):
    """q and out as slices of wider buffers."""
    c = paged_case(10, 2, 64, dt, [70, 400], [1, 33], 32, 50, seed=6)
    T = c["q"].shape[0]
    wide = torch.zeros((T, 3, 10, 64), dtype=dt, device="cuda")
    wide[:, 1] = c["q"]
    want = run_paged(c)
    c["q"] = wide[:, 1]
    out = torch.zeros((T, 10, 2, 64), dtype=dt, device="cuda")
    run_paged(c, out=out[:, :, 1])
    n = c["cu_host"][-1]
    assert torch.equal(out[:n, :, 1], want[:n]) and not bool(out[:, :, 0].any())


def test_paged_scores_that_are_all_minus_infinity():
    """-Inf in every key a row sees: no softmax exists, NaN; in some of them: weight 0."""
    c = paged_case(2, 2, 64, BF16, [40, 40], [1, 1], 16, 0, seed=8)
    q, k = c["q"], c["k"]
    q[:2] = 1.0
    k[c["table"][0].long(), :, 0] = -math.inf
    k[c["table"][0, 2].long(), 8:, 0] = math.nan
    rows = c["table"][1].long()
    k[rows[0], :, 1] = -math.inf
    c["keys"] = [(c["k"][c["table"][s].long()].reshape(-1, 2, 64)[:40], c["v"][c["table"][s].long()].reshape(-1, 2, 64)[:40])
                 for s in range(2)]
    got = run_paged(c)
    assert bool(torch.isnan(got[0, 0]).all())
    o, _, m = attend(q[1:2], *c["keys"][1], torch.tensor([40]), 64 ** -0.5)
    check(got[1:2], o, m, BF16)
    o, _, m = attend(q[:1, 1:], c["keys"][0][0][:, 1:], c["keys"][0][1][:, 1:], torch.tensor([40]), 64 ** -0.5)
    check(got[:1, 1:], o, m, BF16)


def test_paged_a_value_that_is_not_finite():
    c = paged_case(10, 2, 128, F16, [300, 300], [40, 1], 16, 64, seed=9)
    page = c["table"][0, 280 // 16].long()
    c["v"][page, 280 % 16, 1, 5] = math.nan
    c["keys"][0][1][280, 1, 5] = math.nan
    n = c["cu_host"][-1]
    o, _, m = paged_ref(c)
    check(run_paged(c)[:n], o, m, F16)


def test_paged_on_another_stream():
    c = paged_case(40, 8, 128, BF16, [3000, 200], [1, 1], 16, 500, seed=10)
    want = run_paged(c)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    outs = [run_paged(c, stream=s) for _ in range(4)]
    s.synchronize()
    assert all(torch.equal(o[:2], want[:2]) for o in outs)  # rows 2 and 3 belong to no sequence


@pytest.mark.parametrize("prefix", [0, 300])
def test_paged_captured_call_follows_its_lengths(prefix):
    """A captured step replayed with longer sequences, other pages and other queries."""
    c = paged_case(10, 2, 128, F16, [600, 900, 17], [1] * 3, 16, prefix, seed=11, poison=False)
    n = 3
    out = torch.zeros_like(c["q"])
    lens = c["lens"].clone()
    kw = dict(max_kv_len=1000, out=out)
    c["lens"].fill_(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_paged(c, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_paged(c, **kw)
    for new in (lens, lens // 2 + 1):
        c["lens"].copy_(new)
        c["q"].normal_()
        graph.replay()
        torch.cuda.synchronize()
        full = c["keys"]
        c["keys"] = [(k[: int(m)], v[: int(m)]) for (k, v), m in zip(full, new)]
        o, _, m = paged_ref(c)
        c["keys"] = full
        check(out[:n], o, m, F16)


def test_two_captured_calls_replayed_at_once():
    """Two graphs, each with its own workspace, on two streams."""
    cs = [paged_case(40, 8, 128, BF16, [2000, 1500], [1, 1], 16, 200, seed=20 + i) for i in range(2)]
    want = [run_paged(c) for c in cs]
    graphs, outs = [], [torch.zeros_like(c["q"]) for c in cs]
    for c, out in zip(cs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run_paged(c, out=out)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out[:2], w[:2])


def test_bad_numbers_are_reported_and_touch_nothing():
    """Page numbers, lengths and offsets out of range: the call skips them and says so; other sequences are right."""
    for rows in ([1, 1, 1], [1, 30, 1]):
        c = paged_case(10, 2, 128, F16, [40, 100, 50], rows, 16, 0, seed=12)
        o, _, m = paged_ref(c)
        good = c["table"].clone(), c["lens"].clone(), c["cu"].clone()
        n0, n1, n2, n3 = c["cu_host"]
        for bad in (-1, 10 ** 9, c["k"].shape[0]):
            c["table"][1, 2] = bad
            got = run_paged(c)
            with pytest.raises(_lib.HQError, match="HQ_ERR_BAD_INDEX"):
                hq.check_device_error()
            check(got[n0:n1], o[n0:n1], m[n0:n1], F16), check(got[n2:n3], o[n2:n3], m[n2:n3], F16)
            c["table"].copy_(good[0])
        for bad in (-5, 2 ** 30):
            c["lens"][1] = bad
            out = torch.full_like(c["q"], 7.0)
            got = run_paged(c, out=out)
            with pytest.raises(_lib.HQError, match="HQ_ERR_BAD_INDEX"):
                hq.check_device_error()
            check(got[n0:n1], o[n0:n1], m[n0:n1], F16), check(got[n2:n3], o[n2:n3], m[n2:n3], F16)
            c["lens"].copy_(good[1])
        c["cu"][-1] = 10 ** 6
        got = run_paged(c)
        with pytest.raises(_lib.HQError, match="HQ_ERR_BAD_INDEX"):
            hq.check_device_error()
        check(got[n0:n1], o[n0:n1], m[n0:n1], F16), check(got[n1:n2], o[n1:n2], m[n1:n2], F16)
        c["cu"].copy_(good[2])
        check(run_paged(c)[:n3], o, m, F16)
        hq.check_device_error()


@pytest.mark.parametrize("causal", [True, False])
def test_a_long_prompt(causal):
    """40000 tokens; rows at the begin, in the middle and at the end."""
    T, D = 40000, 64
    q, k, v = qkv_rows(T, 2, 1, D, BF16, gen(31))
    got = at.attn_prompt(q, k, v, torch.tensor([0, T], dtype=torch.int32, device="cuda"), T, causal=causal)
    for a in (0, 19990, T - 64):
        seen = torch.arange(a + 1, a + 65) if causal else torch.full((64,), T)
        o, _, m = attend(q[a: a + 64], k, v, seen, D ** -0.5)
        check(got[a: a + 64], o, m, BF16)


def test_a_bound_of_the_prompts_that_is_wrong():
    """max_seqlen sizes the launch only."""
    q, k, v = qkv_rows(700, 10, 2, 128, F16, gen(32))
    cu = torch.tensor([0, 600, 700], dtype=torch.int32, device="cuda")
    o, _, m = prompt_ref(q, k, v, [0, 600, 700], 128 ** -0.5)
    for bound in (0, 1, 600, 10 ** 6):
        check(at.attn_prompt(q, k, v, cu, bound), o, m, F16)


def test_row_offsets_past_32_bits():
    """q, k, v and out as columns of rows 2^20 elements apart."""
    T, Hq, Hk, D = 2300, 4, 2, 64
    wide = torch.zeros((T, 1 << 20), dtype=F16, device="cuda")  # 2.4e9 elements
    base = torch.randn((T, 16, D), generator=gen(33), device="cuda", dtype=F16)
    part = wide[:, : 16 * D].view(T, 16, D)
    part.copy_(base)
    q, k, v, out = part[:, :4], part[:, 4:6], part[:, 6:8], part[:, 8:12]
    cu = torch.tensor([0, 5, T], dtype=torch.int32, device="cuda")
    at.attn_prompt(q, k, v, cu, T, out=out)
    seen = torch.arange(T - 5 - 100 + 1, T - 5 + 1)
    o, _, m = attend(q[T - 100:], k[5:], v[5:], seen, D ** -0.5)
    check(out[T - 100:], o, m, F16)
    assert torch.equal(part[:, :8], base[:, :8]) and torch.equal(part[:, 12:], base[:, 12:])


def test_captured_prompts_follow_their_offsets():
    """A captured call replayed with other prompts in the same rows."""
    T, Hq, Hk, D = 900, 10, 2, 128
    q, k, v = qkv_rows(T, Hq, Hk, D, BF16, gen(30))
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    out = torch.zeros((T, Hq, D), dtype=BF16, device="cuda")
    at.attn_prompt(q, k, v, cu, T, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        at.attn_prompt(q, k, v, cu, T, out=out)
    for new in ([0, 900, 900, 900], [0, 300, 301, 800], [0, 0, 0, 0], [0, 17, 400, 900]):
        cu.copy_(torch.tensor(new, dtype=torch.int32))
        q.normal_()
        out.fill_(7.0)
        graph.replay()
        o, _, m = prompt_ref(q, k, v, new, D ** -0.5)
        check(out[: new[-1]], o, m, BF16)
        assert bool((out[new[-1]:] == 7).all())


def test_calls_on_two_streams_at_once():
    """Eager calls without a workspace of the caller's, on two streams: each has its own."""
    cs = [paged_case(40, 8, 128, F16, [2000 + i, 1500, 700], [1, 1, 70], 16, 300, seed=40 + i) for i in range(2)]
    q, k, v = qkv_rows(1100, 32, 4, 128, BF16, gen(42))
    cu = torch.tensor([0, 1100], dtype=torch.int32, device="cuda")
    want = [run_paged(c) for c in cs] + [at.attn_prompt(q, k, v, cu, 1100)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(8):
        got += [run_paged(c, stream=s) for c, s in zip(cs, streams)]
        got.append(at.attn_prompt(q, k, v, cu, 1100, stream=streams[2]))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        n = cs[i % 3]["cu_host"][-1] if i % 3 < 2 else 1100
        assert torch.equal(g[:n], want[i % 3][:n])


def test_workspaces():
    """What the size call asks for suffices; less, none and a misaligned one are refused."""
    c = paged_case(10, 2, 128, F16, [3000, 9000], [1, 30], 16, 300, seed=50)
    T, n = c["q"].shape[0], c["cu_host"][-1]
    shape = at._SHAPE(T, 2, 30, 10, 2, 128, _lib.HQ_F16, 1.0)
    need = _lib.lib().hq_attn_paged_workspace_size(shape, 9000, 300)
    assert need > 0
    want = run_paged(c, max_kv_len=9000)
    ws = torch.full((need + 16,), 0xFF, dtype=torch.uint8, device="cuda")  # its first contents do not matter
    assert torch.equal(run_paged(c, max_kv_len=9000, workspace=ws[:need])[:n], want[:n])
    for bad, name in ((ws[: need - 1], "WORKSPACE_TOO_SMALL"), (ws[8:], "MISALIGNED"), (ws[:0], "INVALID_ARG|TOO_SMALL")):
        with pytest.raises(_lib.HQError, match=name):
            run_paged(c, max_kv_len=9000, workspace=bad)
    with pytest.raises(_lib.HQError, match="on device"):
        run_paged(c, max_kv_len=9000, workspace=torch.empty(need, dtype=torch.uint8))


def test_more_rows_than_announced():
    """A sequence of more rows than max_q_len is left out and reported where the launch has no kernel for it; the
    others are right."""
    c = paged_case(10, 2, 128, F16, [40, 100, 50], [1, 3, 1], 16, 0, seed=51)
    o, _, m = paged_ref(c)
    c["max_q"] = 1
    got = run_paged(c, out=torch.full_like(c["q"], 7.0))
    with pytest.raises(_lib.HQError, match="HQ_ERR_BAD_INDEX"):
        hq.check_device_error()
    assert bool((got[1:4] == 7).all())
    check(got[:1], o[:1], m[:1], F16), check(got[4:5], o[4:5], m[4:5], F16)


def test_bad_offsets_of_prompts_are_reported():
    q, k, v = qkv_rows(300, 10, 2, 128, F16, gen(52))
    o, _, m = prompt_ref(q, k, v, [0, 100], 128 ** -0.5)
    for bad in ([0, 100, 301], [0, 100, 50], [0, 100, -4], [0, 100, 2 ** 31 - 1]):
        out = torch.full_like(q, 7.0)
        at.attn_prompt(q, k, v, torch.tensor(bad, dtype=torch.int32, device="cuda"), 300, out=out)
        with pytest.raises(_lib.HQError, match="HQ_ERR_BAD_INDEX"):
            hq.check_device_error()
        check(out[:100], o, m, F16)
        assert bool((out[100:] == 7).all())


def test_cache_offsets_past_32_bits():
    """Pages more than 2^32 bytes, and more than 2^31 elements, from the start of the cache."""
    num, page, Hk, D = 70000, 16, 16, 128  # 2.3e9 elements, 4.6 GB
    k = torch.zeros((num, page, Hk, D), dtype=F16, device="cuda")
    v = torch.zeros_like(k)
    g = gen(13)
    T, n = 2, 500
    pages = torch.arange(num - 32, num, device="cuda", dtype=torch.int32)
    kk, vv = (torch.randn((n, Hk, D), generator=g, device="cuda", dtype=F16) for _ in range(2))
    table = torch.stack([pages, pages.flip(0)])
    lens = torch.tensor([n, 1], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n, n], dtype=torch.int32, device="cuda")
    at.kv_append(kk, vv, k, v, table, lens, cu)
    q = torch.randn((1, Hk, D), generator=g, device="cuda", dtype=F16)
    for rows in (1, 40):
        qq = torch.randn((rows, Hk, D), generator=g, device="cuda", dtype=F16)
        got = at.attn_paged(qq, k, v, table[:1], lens[:1], torch.tensor([0, rows], dtype=torch.int32, device="cuda"), rows)
        o, _, m = attend(qq, kk, vv, torch.arange(n - rows + 1, n + 1), D ** -0.5)
        check(got, o, m, F16)
    hq.check_device_error()
