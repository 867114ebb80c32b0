"""Cache kernels: rows into pages and pages over pages, byte for byte; the pool, the cache and attention together."""
import random

import pytest
import torch

from attn_ref import attend, check
from nebula_b200 import _lib, hq
from nebula_b200 import attention as at

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("Hk,D,dt,page,lens,rows", [
    (8, 128, BF16, 16, [777], [1]),
    (1, 8, F16, 16, [1, 16, 17, 0], [1, 16, 2, 0]),
    (2, 96, F16, 32, [500, 33, 64], [1, 33, 40]),
    (16, 64, BF16, 64, [1000] * 9, [1000] * 9),
    (8, 128, F16, 16, list(range(1, 301)), [1] * 300),
    (40, 128, BF16, 256, [70, 300], [70, 5]),
    (5, 8, F16, 16, [40, 3], [9, 3]),
    (3, 40, BF16, 16, [100], [37]),
    (7, 120, F16, 32, [0, 65], [0, 65]),
])
def test_append(Hk, D, dt, page, lens, rows, layout):
    g = torch.Generator(device="cuda").manual_seed(1)
    used = [-(-n // page) for n in lens]
    num = sum(used) + 1
    shape = (num, page, Hk, D) if layout == "nhd" else (num, Hk, page, D)
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=dt) for _ in range(2))
    if layout == "hnd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    perm = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(used + [1])), -1, dtype=torch.int32, device="cuda")
    want_k, want_v = k.clone(), v.clone()
    T = sum(rows) + 2
    wide = torch.randn((T, 2, Hk, D), generator=g, device="cuda", dtype=dt)
    nk, nv = wide[:, 0], wide[:, 1]
    i = r = 0
    for s, (n, m) in enumerate(zip(lens, rows)):
        mine = perm[i: i + used[s]]
        table[s, : used[s]] = mine
        i += used[s]
        where = torch.arange(n - m, n, device="cuda")
        want_k[mine[where // page].long(), where % page] = nk[r: r + m]
        want_v[mine[where // page].long(), where % page] = nv[r: r + m]
        r += m
    cu = torch.tensor([sum(rows[:s]) for s in range(len(rows) + 1)], dtype=torch.int32, device="cuda")
    at.kv_append(nk, nv, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    hq.check_device_error()


def test_append_skips_and_reports_what_has_no_place():
    k, v = torch.zeros((4, 16, 2, 64), device="cuda", dtype=F16), torch.zeros((4, 16, 2, 64), device="cuda", dtype=F16)
    new = torch.ones((3, 2, 64), device="cuda", dtype=F16)
    I = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for table, lens in ((I(4, 1, 2), I(1, 1, 1)), (I(-1, 1, 2), I(1, 1, 1)), (I(0, 1, 2), I(0, 1, 1)), (I(0, 1, 2), I(17, 1, 1)),
                        (I(0, 1, 2), I(-3, 1, 1))):
        k.zero_(), v.zero_()
        at.kv_append(new, new, k, v, table[:, None], lens)
        with pytest.raises(_lib.HQError, match="HQ_ERR_BAD_INDEX"):
            hq.check_device_error()
        assert bool((k[1:3, 0] == 1).all()) and float(k.sum()) == float(v.sum()) == 2 * 128
    hq.check_device_error()


@pytest.mark.parametrize("layers,num,page,Hk,D,n", [(0, 4, 16, 1, 8, 1), (3, 64, 16, 2, 96, 20), (40, 700, 16, 1, 64, 300),
                                                     (2, 3000, 16, 1, 8, 1500)])
def test_copy_pages(layers, num, page, Hk, D, n):
    g = torch.Generator(device="cuda").manual_seed(2)
    shape = (num, page, Hk, D) if layers == 0 else (layers, num, page, Hk, D)
    pools = [torch.randn(shape, generator=g, device="cuda", dtype=BF16) for _ in range(2)]
    order = list(range(num))
    random.Random(n).shuffle(order)
    dst, src = order[:n], [order[n + i % max(1, (num - n) // 2)] for i in range(n)]
    want = [p.clone() for p in pools]
    for p, w in zip(pools, want):
        d, s = torch.tensor(dst, device="cuda"), torch.tensor(src, device="cuda")
        if layers:
            w[:, d] = p[:, s]
        else:
            w[d] = p[s]
    at.kv_copy_pages(pools, src, dst)
    assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_copy_pages_of_interleaved_and_head_first_pools():
    both = torch.randn((9, 2, 4, 16, 64), device="cuda", dtype=F16)
    want = both.clone()
    want[5], want[2, 1] = both[3], both[3, 1]
    at.kv_copy_pages([both[:, 0].transpose(1, 2)], [3], [5])
    at.kv_copy_pages([both[:, 1].transpose(1, 2)], [3, 3], [5, 2])
    assert torch.equal(both, want)


def test_on_another_stream():
    """Append, copy and attention on a stream that is not the current one, one behind the other."""
    g = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.zeros((64, 16, 2, 64), device="cuda", dtype=F16) for _ in range(2))
    nk, nv, q = (torch.randn((500, h, 64), generator=g, device="cuda", dtype=F16) for h in (2, 2, 10))
    table = torch.arange(32, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([500], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 500], dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    at.kv_append(nk, nv, k, v, table, lens, cu, stream=s)
    at.kv_copy_pages([k, v], range(32), range(32, 64), stream=s)
    got = at.attn_paged(q, k, v, table + 32, lens, cu, 500, stream=s)
    s.synchronize()
    o, _, mag = attend(q, nk, nv, torch.arange(1, 501), 64 ** -0.5)
    check(got, o, mag, F16)
    assert torch.equal(k[32:], k[:32]) and torch.equal(v[32:], v[:32])


def test_copy_pages_in_a_captured_call():
    pool = torch.randn((8, 16, 2, 64), device="cuda", dtype=F16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        at.kv_copy_pages([pool], [0, 1], [6, 7])
    pool[:2].fill_(3.0)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((pool[6:] == 3).all())


def test_cache_life_of_a_few_sequences():
    """Prompts, decode steps, forks that write on, frees and compactions: after every step the attention of every
    sequence equals that over a plain list of its keys."""
    Hq, Hk, D, page, layers = 10, 2, 64, 16, 2
    cache = at.KVCache(layers, 40, page, Hk, D, dtype=F16)
    g = torch.Generator(device="cuda").manual_seed(5)
    r = random.Random(5)
    plain = {}  # sequence -> per layer (k, v)

    def rnd(*s):
        return torch.randn(s, generator=g, device="cuda", dtype=F16)

    def step(seqs, counts):
        cache.extend(seqs, counts)
        table, lens, longest = cache.tables(seqs)
        cu = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
        T = sum(counts)
        for layer in range(layers):
            q, k, v = rnd(T, Hq, D), rnd(T, Hk, D), rnd(T, Hk, D)
            at.kv_append(k, v, cache.k[layer], cache.v[layer], table, lens, cu)
            got = at.attn_paged(q, cache.k[layer], cache.v[layer], table, lens, cu, max(counts), max_kv_len=longest)
            a = 0
            for s, n in zip(seqs, counts):
                pk, pv = plain[s][layer]
                plain[s][layer] = pk, pv = torch.cat([pk, k[a: a + n]]), torch.cat([pv, v[a: a + n]])
                m = pk.shape[0]
                o, _, mag = attend(q[a: a + n], pk, pv, torch.arange(m - n + 1, m + 1), D ** -0.5)
                check(got[a: a + n], o, mag, F16)
                a += n

    for i in range(40):
        what = r.choice(["new", "step", "step", "fork", "free", "compact"])
        if what == "new" and len(plain) < 5 and cache.pool.free_pages > 10:
            s = cache.new_seq()
            plain[s] = [(rnd(0, Hk, D), rnd(0, Hk, D)) for _ in range(layers)]
            step([s], [r.randint(1, 60)])
        elif what == "fork" and plain and len(plain) < 6:
            s = r.choice(sorted(plain))
            plain[cache.fork(s)] = list(plain[s])
        elif what == "free" and len(plain) > 2:
            s = r.choice(sorted(plain))
            cache.free(s)
            del plain[s]
        elif what == "compact":
            cache.compact()
        if plain and cache.pool.free_pages > 3 * len(plain):
            step(sorted(plain), [r.choice([1, 1, 1, 20]) for _ in plain])
    hq.check_device_error()
    assert len(plain) > 1
