"""Attention at the limits of its arguments, on the device."""
import pytest

from attn_ref import check
from nebula_b200 import hq
from test_gpu_attn import BF16, F16, paged_case, paged_ref, run_paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hk,D,dt", [(5, 1, 128, F16), (64, 1, 64, BF16), (17, 1, 128, BF16), (40, 8, 128, F16)])
@pytest.mark.parametrize("lens", [[300], [20, 3000, 1]])
@pytest.mark.parametrize("prefix", [0, 60])
def test_a_bound_of_no_rows(Hq, Hk, D, dt, lens, prefix):
    """max_q_len = 0 where every sequence has one: computed, not left out in silence."""
    c = paged_case(Hq, Hk, D, dt, lens, [1] * len(lens), 16, prefix, seed=60 + Hq)
    c["max_q"] = 0
    o, _, m = paged_ref(c)
    check(run_paged(c)[: len(lens)], o, m, dt)
    hq.check_device_error()
