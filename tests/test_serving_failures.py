"""What a failed call of the batcher or of the cache leaves behind, on the host."""
import ctypes

import numpy as np
import pytest
import torch

from nebula_b200 import _lib
from nebula_b200.batcher import SplitFuseBatcher
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
