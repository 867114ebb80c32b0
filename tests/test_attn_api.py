"""Attention and cache entry points without a device: refusals, the index checks that the kernels share, the pool."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest
import torch

from nebula_b200 import _lib
from nebula_b200 import attention as at

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16 = torch.float16
P = 0x10000  # an aligned address that no refused call follows


class Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("stride_token", ctypes.c_int64), ("stride_head", ctypes.c_int64)]


class Pages(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("stride_page", ctypes.c_int64), ("stride_token", ctypes.c_int64),
                ("stride_head", ctypes.c_int64)]


class Shape(ctypes.Structure):
    _fields_ = [("n_tokens", ctypes.c_int), ("n_seqs", ctypes.c_int), ("max_q_len", ctypes.c_int),
                ("n_heads", ctypes.c_int), ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("dtype", ctypes.c_int), ("scale", ctypes.c_float)]


class View(ctypes.Structure):
    _fields_ = [("k", Pages), ("v", Pages), ("num_pages", ctypes.c_int), ("page_size", ctypes.c_int),
                ("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("max_pages", ctypes.c_int),
                ("kv_lens", ctypes.c_void_p)]


def test_packed_structures():
    """The wrappers' packed bytes are the structures of include/hq.h."""
    assert at._ROWS(P, 5, -6) == bytes(Rows(P, 5, -6))
    assert at._SHAPE(1, 2, 3, 4, 5, 6, 1, 0.5) == bytes(Shape(1, 2, 3, 4, 5, 6, 1, 0.5))
    assert at._VIEW(P, 1, 2, 3, P + 16, 4, 5, 6, 7, 16, P + 32, 8, 9, P + 48) == \
        bytes(View(Pages(P, 1, 2, 3), Pages(P + 16, 4, 5, 6), 7, 16, P + 32, 8, 9, P + 48))


def shape(**kw):
    d = dict(n_tokens=4, n_seqs=2, max_q_len=4, n_heads=4, n_kv_heads=2, head_dim=64, dtype=_lib.HQ_F16, scale=0.125)
    d.update(kw)
    return Shape(*d.values())


def rows(p=P, st=256, sh=64):
    return Rows(p, st, sh)


def view(k=P, sp=4096, st=128, sh=64, num=8, page=16, table=P, stride=4, pages=4, lens=P):
    pg = Pages(k, sp, st, sh)
    return View(pg, pg, num, page, table, stride, pages, lens)


def prompt(sh=None, q=None, k=None, v=None, out=None, cu=P):
    r = ctypes.byref
    q, k, v, out = (x or rows() for x in (q, k, v, out))
    return _lib.lib().hq_attn_prompt(r(sh or shape()), r(q), r(k), r(v), cu, 1, r(out), None, None, 0, None)


def paged(sh=None, q=None, c=None, out=None, cu=P, max_kv=64, pt=None, pl=0, ws=P, nb=1 << 30):
    r = ctypes.byref
    return _lib.lib().hq_attn_paged(r(sh or shape()), r(q or rows()), r(c or view()), cu, max_kv, pt, pl, r(out or rows()),
                                    None, ws, nb, None)


@pytest.mark.parametrize("call", [prompt, paged])
def test_refusals_of_shapes_and_rows(call):
    I, U, M = _lib.HQ_ERR_INVALID_ARG, _lib.HQ_ERR_UNSUPPORTED_SHAPE, _lib.HQ_ERR_MISALIGNED
    for kw, status in ((dict(dtype=_lib.HQ_F32), I), (dict(dtype=9), I), (dict(n_tokens=-1), I), (dict(n_seqs=-1), I),
                       (dict(max_q_len=-1), I), (dict(n_kv_heads=0), I), (dict(n_heads=0), U), (dict(n_heads=5), U),
                       (dict(n_heads=129, n_kv_heads=1), U),
                       (dict(head_dim=0), U), (dict(head_dim=12), U), (dict(head_dim=136), U), (dict(scale=0.0), I),
                       (dict(scale=-1.0), I), (dict(scale=float("nan")), I), (dict(scale=float("inf")), I),
                       (dict(n_tokens=1 << 30), U)):
        assert call(shape(**kw)) == status, kw
    for bad, status in ((rows(p=0), I), (rows(p=P + 8), M), (rows(st=100), M), (rows(sh=-64), M)):
        assert call(q=bad) == status and call(out=bad) == status
    # q is read through a tensor map: no broadcast dimension, unless it has one element
    U = _lib.HQ_ERR_UNSUPPORTED_SHAPE
    assert call(q=rows(st=0)) == U and call(q=rows(sh=0)) == U and call(q=rows(st=1 << 40)) == U
    assert call(shape(n_tokens=0)) == _lib.HQ_OK and call(shape(n_seqs=0)) == _lib.HQ_OK  # nothing to do
    assert _lib.lib().hq_last_error_string()


def test_refusals_of_prompts():
    I, M = _lib.HQ_ERR_INVALID_ARG, _lib.HQ_ERR_MISALIGNED
    assert prompt(cu=None) == I
    for bad in (rows(st=0), rows(sh=0), rows(st=1 << 40)):
        assert prompt(k=bad) == prompt(v=bad) == _lib.HQ_ERR_UNSUPPORTED_SHAPE
    for bad, status in ((rows(p=0), I), (rows(p=P + 8), M), (rows(st=100), M)):
        assert prompt(k=bad) == status and prompt(v=bad) == status


def test_refusals_of_caches():
    I, U, M = _lib.HQ_ERR_INVALID_ARG, _lib.HQ_ERR_UNSUPPORTED_SHAPE, _lib.HQ_ERR_MISALIGNED
    r = ctypes.byref

    def append(c=None, k=None, sh=None, cu=P):
        return _lib.lib().hq_kv_append(r(sh or shape()), r(k or rows()), r(rows()), r(c or view()), cu, None)

    for c, status in ((view(k=0), I), (view(k=P + 2), M), (view(sp=100), M), (view(st=4), M), (view(sh=-8), M),
                      (view(page=8), U), (view(page=24), U), (view(page=512), U), (view(num=0), I), (view(pages=-1), I),
                      (view(stride=-1), I), (view(table=None), I), (view(lens=None), I), (view(num=1 << 28), U),
                      (view(pages=1 << 28), U)):
        assert paged(c=c) == status and append(c) == status
    for c in (view(sp=0), view(st=0), view(sh=0)):
        assert paged(c=c) == U
    assert paged(max_kv=-1) == I and paged(pl=-1) == I and paged(pl=5) == I
    assert paged(cu=None, sh=shape(n_seqs=5)) == I and append(cu=None, sh=shape(n_seqs=5)) == I
    assert append(k=rows(p=P + 4)) == M and append(k=rows(p=0)) == I and append(sh=shape(head_dim=4)) == U
    assert append(sh=shape(n_tokens=0)) == _lib.HQ_OK


def test_refusals_of_page_copies():
    I, M = _lib.HQ_ERR_INVALID_ARG, _lib.HQ_ERR_MISALIGNED

    def copy(moves, bases=(P,), stride=4096, size=4096, num=8):
        mv = np.array(moves, np.int32).reshape(-1, 2)
        bs = (ctypes.c_void_p * max(1, len(bases)))(*bases)
        return _lib.lib().hq_kv_copy_pages(bs, len(bases), stride, size, num, mv.ctypes.data, len(mv), None)

    assert copy([]) == _lib.HQ_OK and copy([[0, 1]], bases=()) == _lib.HQ_OK
    for moves in ([[0, 8]], [[-1, 1]], [[8, 1]], [[0, -2]],      # outside the pool
                  [[3, 3]], [[0, 1], [2, 1]],                      # onto itself, written twice
                  [[0, 1], [1, 2]], [[1, 2], [0, 1]]):             # read and written
        assert copy(moves) == I, moves
    assert copy([[0, 1]], bases=(0,)) == I and copy([[0, 1]], bases=(P + 8,)) == M
    assert copy([[0, 1]], size=4090) == M and copy([[0, 1]], stride=4090) == M and copy([[0, 1]], stride=2048) == M
    assert copy([[0, 1]], size=0) == M and copy([[0, 1]], num=0) == I


def test_python_refusals():
    E = _lib.HQError
    q, k = torch.zeros((3, 4, 64), dtype=torch.float16), torch.zeros((3, 2, 64), dtype=torch.float16)
    cu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(E, match="CUDA device"):
        at.attn_prompt(q, k, k, cu, 3)
    with pytest.raises(E, match="unsupported dtype"):
        at.attn_prompt(q.float(), k, k, cu, 3)
    with pytest.raises(E, match="destinations"):
        at.kv_copy_pages([], [1], [])
    for bad in (k[:2], k[:, :1], k[..., :32], k.float()):
        with pytest.raises(E):
            at._rows(bad, "k", F16, -1, (3, 2, 64))
    with pytest.raises(E, match="contiguous"):
        at._rows(torch.zeros((3, 2, 128), dtype=F16)[..., ::2], "k", F16, -1, (3, 2, 64))
    for bad in (cu.long(), cu[:1], torch.zeros(4, dtype=torch.int32)[::2], cu[None]):
        with pytest.raises(E, match="contiguous int32"):
            at._index(bad, "cu", 2, -1)
    pages, table, lens = torch.zeros((5, 16, 2, 64), dtype=torch.float16), torch.zeros((1, 1), dtype=torch.int32), cu[:1]
    at._view(pages, pages, table, lens, F16, -1, 64)
    for bad in ((pages, pages[:4], table, lens), (pages[0], pages[0], table, lens), (pages.float(), pages, table, lens),
                (pages, pages, table[0], lens), (pages, pages, table.long(), lens), (pages, pages, table, cu),
                (pages[..., ::2], pages[..., ::2], table, lens)):
        with pytest.raises(E):
            at._view(*bad, F16, -1, 64)
    for kind in (list, np.array, tuple, lambda x: torch.tensor(x)):
        assert at._moves(kind([3, 4]), kind([7, 1])) == np.array([3, 7, 4, 1], np.int32).tobytes()
    assert at._moves([], []) == b""
    with pytest.raises(E, match="one block"):
        at._page_bytes((16, 2, 64), (256, 64, 1), 2)
    assert at._page_bytes((16, 2, 64), (64, 1024, 1), 2) == 4096
    with pytest.raises(E, match="CUDA device"):
        at.kv_copy_pages([pages], [0], [1])
    with pytest.raises(E, match="no pool"):
        at.PagePool(4, 20)


def test_index_checks(tmp_path):
    """The functions through which the kernels take rows, lengths and page numbers, compiled for the host."""
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include "hq_attn_index.h"
#include <cstdio>
#include <climits>
using namespace hq;
#define CHECK(x) do { if (!(x)) { std::printf("%d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    int f, n;
    const int cu[] = {0, 3, 3, 10, 8, -1, 4, INT_MAX, INT_MIN, INT_MAX};
    CHECK(seq_rows(cu, 0, 10, f, n) && f == 0 && n == 3);
    CHECK(seq_rows(cu, 1, 10, f, n) && n == 0);
    CHECK(seq_rows(cu, 2, 10, f, n) && f == 3 && n == 7);
    CHECK(!seq_rows(cu, 2, 9, f, n));   // past the rows
    CHECK(!seq_rows(cu, 3, 10, f, n));  // falls
    CHECK(!seq_rows(cu, 4, 10, f, n) && !seq_rows(cu, 5, 10, f, n));  // negative
    CHECK(!seq_rows(cu, 6, 10, f, n) && !seq_rows(cu, 7, 10, f, n) && !seq_rows(cu, 8, 10, f, n));
    CHECK(seq_rows(nullptr, 9, 10, f, n) && f == 9 && n == 1 && !seq_rows(nullptr, 10, 10, f, n));
    CHECK(len_ok(0, 0, 16) && len_ok(64, 4, 16) && !len_ok(65, 4, 16) && !len_ok(-1, 4, 16) && !len_ok(INT_MIN, 4, 16));
    CHECK(len_ok(INT_MAX, INT_MAX, 256));
    CHECK(page_ok(0, 1) && !page_ok(1, 1) && !page_ok(-1, 1) && !page_ok(INT_MIN, INT_MAX) && page_ok(INT_MAX - 1, INT_MAX));
    CHECK(keys_seen(10, 3, 0, 1) == 8 && keys_seen(10, 3, 2, 1) == 10 && keys_seen(2, 5, 0, 1) == 0);
    CHECK(keys_seen(2, 5, 2, 1) == 0 && keys_seen(2, 5, 3, 1) == 1 && keys_seen(7, 5, 0, 0) == 7 && keys_seen(0, 1, 0, 1) == 0);
    return 0;
}''')
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "nebula_b200", "csrc"), str(src), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


class PlainPool:
    """The pool's rules with lists: lowest free page first, copy on write of a shared, partly filled last page."""

    def __init__(self, num, page):
        self.num, self.page, self.seqs = num, page, {}

    def refs(self):
        n = [0] * self.num
        for pages, _ in self.seqs.values():
            for g in pages:
                n[g] += 1
        return n

    def free(self):
        return [g for g, n in enumerate(self.refs()) if n == 0]

    def extend(self, s, n):
        pages, length = self.seqs[s]
        copy = n > 0 and length % self.page and self.refs()[pages[-1]] > 1
        want = -(-(length + n) // self.page)
        free = self.free()
        if want - len(pages) + bool(copy) > len(free):
            return None
        moves = []
        if copy:
            moves = [(pages[-1], free[0])]
            pages = pages[:-1] + [free.pop(0)]
        while len(pages) < want:
            pages = pages + [free.pop(0)]
        self.seqs[s] = (pages, length + n)
        return moves


@pytest.mark.parametrize("seed", range(6))
def test_pool_against_plain_lists(seed):
    r = random.Random(seed)
    num, page = r.choice([(5, 16), (40, 16), (200, 32)])
    pool, plain = at.PagePool(num, page), PlainPool(num, page)
    for _ in range(400):
        what = r.choice(["new", "extend", "extend", "extend", "fork", "free", "compact"])
        some = r.choice(sorted(plain.seqs)) if plain.seqs else None
        if what == "new" and len(plain.seqs) < 12:
            s = pool.new_seq()
            assert s not in plain.seqs
            plain.seqs[s] = ([], 0)
        elif what == "fork" and some is not None and len(plain.seqs) < 12:
            s = pool.fork(some)
            assert s not in plain.seqs
            plain.seqs[s] = plain.seqs[some]
        elif what == "free" and some is not None:
            pool.free(some)
            del plain.seqs[some]
            with pytest.raises(_lib.HQError):
                pool.seq_len(some)
        elif what == "extend" and some is not None:
            n = r.choice([0, 1, 1, page - 1, page, r.randint(1, 4 * page)])
            want = plain.extend(some, n)
            if want is None:
                with pytest.raises(_lib.HQError, match="HQ_ERR_OUT_OF_PAGES"):
                    pool.extend(some, n)
            else:
                assert pool.extend(some, n) == want
        elif what == "compact":
            moves = pool.compact()
            live = num - len(plain.free())
            to = dict(moves)
            assert len(to) == len(moves) and all(a >= live > b for a, b in moves)
            assert sorted(to.values()) == [g for g in plain.free() if g < live]
            plain.seqs = {s: ([to.get(g, g) for g in pages], n) for s, (pages, n) in plain.seqs.items()}
        assert pool.free_pages == len(plain.free())
        for s, (pages, n) in plain.seqs.items():
            assert pool.seq_len(s) == n and pool.seq_pages(s).tolist() == list(pages)
        seqs = r.sample(sorted(plain.seqs), r.randint(0, len(plain.seqs)))
        table, lens = pool.tables(seqs)
        assert lens.tolist() == [plain.seqs[s][1] for s in seqs]
        assert table.shape == (len(seqs), max([len(plain.seqs[s][0]) for s in seqs], default=0))
        assert all(row.tolist() == list(plain.seqs[s][0]) + [0] * (table.shape[1] - len(plain.seqs[s][0]))
                   for row, s in zip(table, seqs))
    pool.close()


@pytest.mark.parametrize("seed", range(4))
def test_pool_extends_all_or_none(seed):
    """Several sequences at once, some named twice, are the single extensions in their order, or change nothing."""
    r = random.Random(seed)
    page, num = 16, 12
    refused = 0
    for _ in range(60):
        pool, plain = at.PagePool(num, page), PlainPool(num, page)
        for _ in range(r.randint(1, 6)):
            if plain.seqs and r.random() < 0.6:
                parent = r.choice(sorted(plain.seqs))
                plain.seqs[pool.fork(parent)] = plain.seqs[parent]
            else:
                s = pool.new_seq()
                plain.seqs[s] = ([], 0)
                n = r.randint(0, 2 * page)
                assert pool.extend(s, n) == (plain.extend(s, n) or [])
        seqs = r.choices(sorted(plain.seqs), k=r.randint(0, 8))
        counts = [r.choice([0, 1, 5, page, 2 * page, 4 * page]) for _ in seqs]
        before = dict(plain.seqs), pool.free_pages
        moves = []
        for s, n in zip(seqs, counts):
            m = plain.extend(s, n)
            if m is None:
                plain.seqs, moves = before[0], None
                break
            moves += m
        if moves is None:
            refused += 1
            with pytest.raises(_lib.HQError, match="HQ_ERR_OUT_OF_PAGES"):
                pool.extend(seqs, counts)
        else:
            assert pool.extend(seqs, counts) == moves
        assert pool.free_pages == len(plain.free())
        for s, (pages, n) in plain.seqs.items():
            assert pool.seq_len(s) == n and pool.seq_pages(s).tolist() == list(pages)
        s = pool.new_seq()  # what is free is handed out as before, lowest page first
        assert pool.extend(s, pool.free_pages * page) == [] and pool.seq_pages(s).tolist() == plain.free()
        pool.close()
    assert 0 < refused < 60


def test_pool_refuses_unknown_sequences():
    pool = at.PagePool(4, 16)
    s = pool.new_seq()
    for bad in (-1, s + 1, 10 ** 6):
        for call in (pool.fork, pool.free, pool.seq_len, pool.seq_pages, lambda x: pool.extend(x, 1)):
            with pytest.raises(_lib.HQError):
                call(bad)
    with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
        pool.extend(s, -1)
    for bad in (([s, s], [1]), ([s, s + 1], [1, 1]), ([s, s], [1, -1])):
        with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
            pool.extend(*bad)
    with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
        pool.tables([s, s + 1])
    with pytest.raises(_lib.HQError, match="HQ_ERR_OUT_OF_PAGES"):
        pool.extend(s, 65)
    assert pool.seq_len(s) == 0 and pool.free_pages == 4
    L, n = _lib.lib(), ctypes.c_int(-5)
    assert L.hq_kv_pool_create(0, 16) is None and L.hq_kv_pool_create(1 << 28, 16) is None
    assert L.hq_kv_pool_new_seq(None) == -1 and L.hq_kv_pool_fork(None, 0) == -1 and L.hq_kv_pool_free_pages(None) == 0
    assert L.hq_kv_pool_extend(None, None, None, 0, None, None) == _lib.HQ_ERR_INVALID_ARG
    # a compaction that has no room for its moves changes nothing
    a, b = pool.new_seq(), pool.new_seq()
    pool.extend(a, 16), pool.extend(b, 16)
    pool.free(a)
    assert L.hq_kv_pool_compact(pool._h, None, 0, ctypes.byref(n)) == _lib.HQ_ERR_INVALID_ARG and n.value == -5
    assert pool.seq_pages(b).tolist() == [1] and pool.compact() == [(1, 0)] and pool.compact() == []
    pool.close()
