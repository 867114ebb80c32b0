"""Page, sequence and key numbers that are no whole numbers, or that int32 does not hold, are refused on the host: none
becomes another page or sequence."""
import numpy as np
import pytest
import torch

from nebula_b200 import _lib
from nebula_b200 import attention as at

BIG = 2 ** 32 + 1  # 1 in its lower 32 bits


@pytest.mark.parametrize("bad", [np.array([BIG]), np.array([-BIG]), np.array([2 ** 31]), np.array([BIG], np.uint64),
                                 np.array([3.7]), np.array([1.0], np.float32), np.array(["1"]),
                                 np.array([BIG], object)])
def test_page_moves_of_arrays(bad):
    ok = np.array([2])
    for src, dst in ((bad, ok), (ok, bad)):
        with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
            at._moves(src, dst)
        with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
            at.kv_copy_pages([], src, dst)


def test_page_moves_of_arrays_that_int32_holds():
    for dt in (np.int8, np.uint8, np.int16, np.uint16, np.int32, np.uint32, np.int64, np.uint64):
        assert at._moves(np.array([3, 4], dt), np.array([7, 1], dt)) == np.array([3, 7, 4, 1], np.int32).tobytes()
    top = np.array([2 ** 31 - 1, -2 ** 31])
    assert at._moves(top, top) == np.repeat(top, 2).astype(np.int32).tobytes()
    assert at._moves(np.arange(20)[::5], np.arange(4)[::-1]) == \
        np.array([0, 3, 5, 2, 10, 1, 15, 0], np.int32).tobytes()
    for dt in (np.int64, np.float64):  # np.array([]) is of the latter
        assert at._moves(np.empty(0, dt), np.empty(0, dt)) == b""
    assert at._moves(np.array([True]), np.array([False])) == at._moves([True], [False])
    for bad in ([BIG], [3.7]):
        with pytest.raises((OverflowError, TypeError)):
            at._moves(bad, [1])


@pytest.mark.parametrize("kind", [list, tuple, np.array, torch.tensor, lambda x: x[0]])
def test_sequences_and_counts_of_a_pool(kind):
    pool = at.PagePool(8, 16)
    a, b = pool.new_seq(), pool.new_seq()
    assert pool.extend(kind([b]), kind([17])) == [] and pool.seq_len(b) == 17
    assert pool.tables(kind([b]))[1].tolist() == [17]
    for bad in (BIG, -BIG, 1.0, 0.5):
        for call in (lambda: pool.extend(kind([bad]), kind([1])), lambda: pool.extend(kind([a]), kind([bad])),
                     lambda: pool.tables(kind([bad]))):
            with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
                call()
    assert pool.seq_len(a) == 0 and pool.seq_len(b) == 17 and pool.free_pages == 6
    assert pool.extend([], []) == [] and pool.tables([])[0].shape == (0, 0)
    pool.close()


def test_a_sequence_of_a_pool():
    pool = at.PagePool(8, 16)
    a, b = pool.new_seq(), pool.new_seq()
    pool.extend(b, 17)
    for bad in (BIG, -BIG + 2, 2 ** 31, 1.0):
        for call in (pool.fork, pool.free, pool.seq_len, pool.seq_pages):
            with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
                call(bad)
    assert pool.seq_len(np.int64(b)) == 17 and pool.free_pages == 6
    pool.free(np.int32(b))
    assert pool.free_pages == 8
    pool.close()


def test_sizes_of_a_pool():
    for size in ((2 ** 32 + 4, 16), (4, 2 ** 32 + 16), (4.0, 16), (4, 16.0)):
        with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
            at.PagePool(*size)


@pytest.mark.parametrize("dt", [np.int32, np.int64])
def test_sequences_and_counts_in_strided_arrays(dt):
    """Every second element, in either order: the numbers that the array shows, not those that lie beside them."""
    pool = at.PagePool(20, 16)
    seqs = np.array([pool.new_seq() for _ in range(6)], dt)
    counts = np.array([1, 20, 3, 40, 5, 60], dt)
    pool.extend(seqs[::2], counts[::2])
    pool.extend(seqs[::-2], counts[::-2])
    assert [pool.seq_len(int(s)) for s in seqs] == counts.tolist()
    table, lens = pool.tables(seqs[::-1])
    assert lens.tolist() == counts[::-1].tolist()
    assert [row[0] for row in table] == [pool.seq_pages(int(s))[0] for s in seqs[::-1]]
    both = np.stack([seqs, counts], 1)  # columns
    pool.extend(both[:, 0], both[:, 1])
    assert pool.tables(both[:, 0])[1].tolist() == (2 * counts).tolist()
    pool.close()
