"""What a failed call of the batcher or of the cache leaves behind, on the host."""
import ctypes

import numpy as np
import pytest
import torch

from nebula_b200 import _lib
from nebula_b200.batcher import COMPLETED, SplitFuseBatcher
from test_serving import HostCache, keys, write


def test_a_fork_that_fails_submits_nothing():
    cache = HostCache(8, 16)
    b = SplitFuseBatcher(cache=cache)
    parent = b.submit_request(20, 4)
    b.plan_attention(b.assemble_step_batch())
    cache.free(b._seqs[parent][0])  # behind the batcher's back
    with pytest.raises(_lib.HQError, match="no sequence"):
        b.submit_request(3, 4, parent)
    assert b.num_active_requests() == 1 and list(b._seqs) == [parent]
    with pytest.raises(_lib.HQError):
        b.request_state(parent + 1)
    del b._seqs[parent]
    b.close()


def test_a_request_that_is_refused_forks_nothing():
    cache = HostCache(8, 16)
    b = SplitFuseBatcher(cache=cache)
    parent = b.submit_request(20, 4)
    b.plan_attention(b.assemble_step_batch())
    with pytest.raises(ctypes.ArgumentError):
        b.submit_request(3.5, 4, parent)
    assert b.num_active_requests() == 1 and cache.new_seq() == 1  # the number after the parent's: no fork has it
    b.close()


class FailingCache(HostCache):
    """Its next `failures` copies of pages raise."""
    failures = 0

    def _copy(self, moves, stream):
        if moves and self.failures:
            self.failures -= 1
            raise RuntimeError("no copy")
        super()._copy(moves, stream)


def marked(cache, n):
    """A sequence of n keys with the marks 1 .. n."""
    s = cache.new_seq()
    cache.extend([s], [n])
    for j, (page, slot) in enumerate((p, i) for p in cache.pool.seq_pages(s) for i in range(cache.pool.page_size)):
        if j < n:
            cache.k[0, int(page), slot, 0, 0] = j + 1.0
    return s


@pytest.mark.parametrize("again", ["same", "nothing", "other", "compact"])
def test_copies_that_fail_are_made_by_the_next_call(again):
    """The pool has moved on by then: the copy is owed, not lost."""
    cache = FailingCache(9, 16)
    a = marked(cache, 21)
    b, other = cache.fork(a), marked(cache, 3)
    cache.failures = 1
    with pytest.raises(RuntimeError, match="no copy"):
        cache.extend([b], [2])
    assert cache.pool.seq_len(b) == 23 and cache.pool.seq_pages(a)[1] != cache.pool.seq_pages(b)[1]
    if again == "compact":
        cache.free(other)
        cache.compact()
    else:
        cache.extend(*{"same": ([b], [0]), "nothing": ([], []), "other": ([other], [1])}[again])
    for s in (a, b):
        assert keys(cache, cache.pool.seq_pages(s), 21) == [j + 1.0 for j in range(21)]


def test_a_compaction_that_fails_is_made_up_for():
    cache = FailingCache(9, 16)
    a, b = marked(cache, 40), marked(cache, 21)
    c = cache.fork(b)
    cache.free(a)
    cache.failures = 3
    for call in (cache.compact, lambda: cache.extend([c], [1]), cache.compact):  # owed in turn: moved, copied, moved
        with pytest.raises(RuntimeError, match="no copy"):
            call()
    cache.extend([], [])
    for s in (b, c):
        assert keys(cache, cache.pool.seq_pages(s), 21) == [j + 1.0 for j in range(21)]


def test_a_closed_batcher_gives_its_pages_back():
    cache = HostCache(8, 16)
    b = SplitFuseBatcher(cache=cache)
    parent = b.submit_request(20, 4)
    b.plan_attention(b.assemble_step_batch())
    b.submit_request(3, 4, parent)
    assert cache.pool.free_pages == 6
    b.close()
    assert cache.pool.free_pages == 8 and not b._seqs
    b.close()
    cache.pool.close()  # before its batcher: nothing to give back to
    b = SplitFuseBatcher(cache=HostCache(8, 16))
    b.submit_request(20, 4)
    b.plan_attention(b.assemble_step_batch())
    b.cache.pool.close()
    b.close()


@pytest.mark.parametrize("q,k,v", [(3, 4, 4), (4, 3, 4), (4, 3, 3), (4, 4, 3), (4, 0, 0)])
def test_attend_takes_the_rows_of_its_step(q, k, v):
    """With too few keys the last sequences would attend to what their pages held before."""
    b = SplitFuseBatcher(cache=HostCache(3, 16))
    b.submit_request(4, 4)
    step = b.plan_attention(b.assemble_step_batch())
    with pytest.raises(ValueError, match="rows for a step of 4"):
        b.attend(step, 0, *[torch.zeros((n, 1, 8), dtype=torch.float16) for n in (q, k, v)])
    b.close()


class Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


def test_a_steps_copies_and_attention_are_of_one_stream():
    """The copy of a page that a fork shares is made on the plan's stream, and attend refuses another."""
    class Cache(HostCache):
        def _copy(self, moves, stream):
            if moves:
                self.on = stream
            super()._copy(moves, stream)

    cache = Cache(8, 16)
    b = SplitFuseBatcher(cache=cache)
    parent = b.submit_request(20, 4)
    batch = b.assemble_step_batch()
    b.plan_attention(batch)
    b.update_step_completion(batch)
    b.submit_request(3, 4, parent)
    mine, same, other = Stream(7), Stream(7), Stream(8)
    step = b.plan_attention(b.assemble_step_batch(), stream=mine)
    assert cache.on is mine and step.stream is mine
    rows = [torch.zeros((step.rows, 1, 8), dtype=torch.float16)] * 3
    with pytest.raises(ValueError, match="another stream"):
        b.attend(step, 0, *rows, stream=other)
    for ok in (None, mine, same):
        with pytest.raises(_lib.HQError, match="CUDA device"):  # the host's cache comes no further
            b.attend(step, 0, *rows, stream=ok)
    b.close()


def test_a_request_given_up_makes_room_for_the_others():
    """A step without pages: one request leaves, its pages with it, and the step goes on."""
    cache = HostCache(3, 16)
    b = SplitFuseBatcher(16, 16, 64, cache=cache)
    a, c = b.submit_request(30, 4), b.submit_request(16, 9)
    for _ in range(3):
        batch = b.assemble_step_batch()
        b.plan_attention(batch)
        b.update_step_completion(batch)
    old = b.assemble_step_batch()
    with pytest.raises(_lib.HQError, match="HQ_ERR_OUT_OF_PAGES"):
        b.plan_attention(old)
    b.cancel_request(a)
    assert cache.pool.free_pages == 2 and b.num_active_requests() == 1
    assert b.request_state(a)["status"] == COMPLETED and b.request_state(a)["decode_tokens_generated"] == 1
    with pytest.raises(ValueError, match=f"request {a} is not active"):
        b.plan_attention(old)  # a batch from before
    with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
        b.cancel_request(a)
    batch = b.assemble_step_batch()
    assert [x.request_id for x in batch.chunks] == [c]
    while b.has_active_work():
        batch = b.assemble_step_batch()
        b.plan_attention(batch)
        b.update_step_completion(batch)
    assert cache.pool.free_pages == 3
    b.close()


def test_requests_given_up_at_any_stage():
    """Queued, in prefill, decoding; children keep the shared keys; a batch assembled before completes the others only."""
    cache = HostCache(20, 16)
    b = SplitFuseBatcher(16, 16, 64, cache=cache)
    first, second, third = b.submit_request(40, 9), b.submit_request(5, 9), b.submit_request(5, 2)
    for bad in (0, 4, 99, -1, 2 ** 32 + 1):
        with pytest.raises(_lib.HQError, match="HQ_ERR_INVALID_ARG"):
            b.cancel_request(bad)
    batch = b.assemble_step_batch()
    write(cache, b.plan_attention(batch), range(1, 17))
    child = b.submit_request(1, 1, first)
    b.cancel_request(second)  # queued
    b.cancel_request(first)   # in prefill, in a batch
    b.update_step_completion(batch)
    assert b.request_state(first)["prefill_completed_tokens"] == 0 and b.num_active_requests() == 2
    batch = b.assemble_step_batch()
    assert [x.request_id for x in batch.chunks] == [third]
    b.plan_attention(batch)
    b.update_step_completion(batch)
    batch = b.assemble_step_batch()
    assert [(x.request_id, x.is_prefill) for x in batch.chunks] == [(third, False), (child, True)]
    step = b.plan_attention(batch)
    assert keys(cache, step.page_table[1], 16) == [float(i) for i in range(1, 17)]
    b.cancel_request(third)   # decoding, in a batch
    b.update_step_completion(batch)
    batch = b.assemble_step_batch()
    assert [x.request_id for x in batch.chunks] == [child]
    b.plan_attention(batch)
    b.update_step_completion(batch)
    assert not b.has_active_work() and cache.pool.free_pages == 20
    b.reset()
    plain = SplitFuseBatcher()  # without a cache
    n = plain.submit_request(4, 4)
    plain.cancel_request(n)
    assert not plain.has_active_work()
    plain.close()
    b.close()
