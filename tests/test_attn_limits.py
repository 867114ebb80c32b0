"""Limits of attention's sizes on the host: bounds of nought, and lengths next to 2^31."""
import ctypes

import pytest

from nebula_b200 import _lib
from test_attn_api import shape


def size(sh, max_kv, prefix=0):
    return _lib.lib().hq_attn_paged_workspace_size(ctypes.byref(sh), max_kv, prefix)


@pytest.mark.parametrize("heads", [(40, 8), (64, 1), (17, 1), (128, 1)])
@pytest.mark.parametrize("seqs", [1, 3])
def test_a_bound_of_no_rows_plans_as_one_of_one(heads, seqs):
    """A sequence may have more rows than max_q_len, and is reported or computed: a call with a bound of 0 launches what
    one with 1 does, with its workspace."""
    kw = dict(n_tokens=seqs, n_seqs=seqs, n_heads=heads[0], n_kv_heads=heads[1], head_dim=128)
    for max_kv in (100, 20000):
        assert size(shape(max_q_len=0, **kw), max_kv) == size(shape(max_q_len=1, **kw), max_kv)
    assert size(shape(max_q_len=0, **kw), 20000) > 0


@pytest.mark.parametrize("heads,rows", [((40, 8), 1), ((10, 2), 30), ((64, 1), 1), ((8, 8), 4)])
def test_a_bound_of_keys_next_to_the_largest(heads, rows):
    """max_kv_len is often the longest there can be: it plans as one of a few keys less."""
    for seqs in (1, 70):
        sh = shape(n_tokens=seqs * rows, n_seqs=seqs, max_q_len=rows, n_heads=heads[0], n_kv_heads=heads[1], head_dim=128)
        want = size(sh, 2 ** 31 - 1000)
        assert want > 0
        for bound in (2 ** 31 - 128, 2 ** 31 - 127, 2 ** 31 - 16, 2 ** 31 - 1):
            assert size(sh, bound) == want
