"""The batcher's places in a paged cache, on the host: rows, lengths and pages of every step, sharing, what is freed."""
import random

import pytest
import torch

from nebula_b200 import _lib
from nebula_b200.attention import KVCache
from nebula_b200.batcher import SplitFuseBatcher


class HostCache(KVCache):
    """A cache whose slots hold (request, position) marks: keys of heads 1 and dim 8, moved on the host."""

    def __init__(self, num_pages, page_size):
        super().__init__(1, num_pages, page_size, 1, 8, dtype=torch.float16, device="cpu")

    def _copy(self, moves, stream):
        for pool in (self.k, self.v):
            old = pool.clone()
            for s, d in moves:
                pool[:, d] = old[:, s]


def write(cache, step, rows):
    """What kv_append does; rows: a mark of each row."""
    cu, lens, page = step.cu_q.tolist(), step.kv_lens.tolist(), cache.pool.page_size
    for s in range(len(lens)):
        for i in range(cu[s], cu[s + 1]):
            pos = lens[s] - (cu[s + 1] - i)
            cache.k[0, int(step.page_table[s, pos // page]), pos % page, 0, 0] = rows[i]


def keys(cache, pages, n):
    page = cache.pool.page_size
    return [float(cache.k[0, int(pages[j // page]), j % page, 0, 0]) for j in range(n)]


@pytest.mark.parametrize("seed", range(4))
def test_requests_keep_their_keys(seed):
    r = random.Random(seed)
    cache = HostCache(120, 16)
    prefix = cache.new_seq()
    cache.extend([prefix], [21])
    b = SplitFuseBatcher(24, 16, 64, cache=cache, prefix=prefix)
    want, left, mark = {}, 14, 0.0
    for prompt in (1, 40):
        want[b.submit_request(prompt, 5)] = []
    while b.has_active_work():
        if left and r.random() < 0.4:
            left -= 1
            parent = r.choice([None] + sorted(b._seqs))
            rid = b.submit_request(r.choice([0, 1, 17, 60]), r.randint(0, 9), parent)
            want[rid] = list(want[parent]) if parent else []
        if r.random() < 0.2:
            cache.compact()
        batch = b.assemble_step_batch()
        step = b.plan_attention(batch)
        if r.random() < 0.2:  # a plan made again is the same plan
            again = b.plan_attention(batch)
            assert all(torch.equal(getattr(step, f), getattr(again, f)) for f in ("cu_q", "page_table", "kv_lens"))
        chunks = [c for c in batch.chunks if c.num_tokens]
        assert step.rows == batch.total_batch_tokens == int(step.cu_q[-1])
        assert step.cu_q.diff().tolist() == [c.num_tokens for c in chunks] and step.prefix_len == 21
        assert step.prefix_table.tolist() == cache.pool.seq_pages(prefix).tolist()
        assert step.max_q_len == max([c.num_tokens for c in chunks], default=0)
        assert step.max_kv_len == max(step.kv_lens.tolist(), default=0)
        marks = [mark + i for i in range(step.rows)]
        mark = (mark + step.rows) % 1900  # float16 holds the integers up to 2048
        write(cache, step, marks)
        for s, c in enumerate(chunks):
            a = int(step.cu_q[s])
            want[c.request_id] += marks[a: a + c.num_tokens]
            assert int(step.kv_lens[s]) == len(want[c.request_id])
        for s, c in enumerate(chunks):
            assert keys(cache, step.page_table[s], len(want[c.request_id])) == want[c.request_id]
        b.update_step_completion(batch)
    assert not b._seqs and cache.pool.free_pages == 120 - 2
    b.close()


def test_a_step_without_pages_changes_nothing():
    cache = HostCache(3, 16)
    b = SplitFuseBatcher(16, 16, 64, cache=cache)
    a, c = b.submit_request(30, 4), b.submit_request(16, 9)
    for _ in range(3):
        batch = b.assemble_step_batch()
        step = b.plan_attention(batch)
        b.update_step_completion(batch)
    assert step.kv_lens.tolist() == [31, 16] and cache.pool.free_pages == 0
    batch = b.assemble_step_batch()  # the second request's 17th key has no page
    for _ in range(2):
        with pytest.raises(_lib.HQError, match="HQ_ERR_OUT_OF_PAGES"):
            b.plan_attention(batch)
        assert [cache.pool.seq_len(b._seqs[x][0]) for x in (a, c)] == [31, 16]
    b.reset()
    assert cache.pool.free_pages == 3 and not b._seqs
    b.close()


def test_refusals():
    b = SplitFuseBatcher()
    b.submit_request(4, 4)
    with pytest.raises(ValueError, match="no cache"):
        b.plan_attention(b.assemble_step_batch())
    with pytest.raises(ValueError, match="holds no keys"):
        b.submit_request(4, 4, parent=1)
    assert b.num_active_requests() == 1
    b.close()
    cache = HostCache(3, 16)
    b = SplitFuseBatcher(cache=cache)
    b.submit_request(4, 4)
    step = b.plan_attention(b.assemble_step_batch())
    with pytest.raises(ValueError, match="3 rows for a step of 4"):
        b.attend(step, 0, *[torch.zeros((3, 1, 8), dtype=torch.float16)] * 3)
    b.close()
