"""Attention at the limits of its arguments, on the device."""
import pytest
import torch

from attn_ref import attend, check
from nebula_b200 import attention as at
from nebula_b200 import hq
from test_gpu_attn import BF16, F16, gen, paged_case, paged_ref, run_paged

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


@pytest.mark.parametrize("prefix", [False, True])
def test_almost_two_to_the_31_keys(prefix):
    """The largest lengths, over few pages that the table names again and again: all scores are 0 but those of the last
    page, about 60, which alone have a weight (2^31 e^-60 is 2e-17)."""
    D, Hq, page, n = 64, 4, 64, 30
    total = 2 ** 31 - 1 if prefix else 2 ** 31 - 64  # a sequence's pages hold at most 2^31 - 1 keys
    k = torch.zeros((6, page, 1, D), device="cuda", dtype=BF16)
    v = torch.randn((6, page, 1, D), generator=gen(70), device="cuda", dtype=BF16)
    q = torch.randn((n, Hq, D), generator=gen(71), device="cuda", dtype=BF16)
    q[:, :, 0] = 8.0
    k[4:] = torch.randn((2, page, 1, D), generator=gen(72), device="cuda", dtype=BF16)
    k[4:, :, :, 0] = 60.0
    table = torch.zeros(-(-total // page), dtype=torch.int32, device="cuda")
    table[1::3], table[2::3], table[-1] = 1, 2, 4
    last = total - (table.shape[0] - 1) * page
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    if prefix:
        lens, own = torch.tensor([page], dtype=torch.int32, device="cuda"), torch.full((1, 1), 5, dtype=torch.int32, device="cuda")
        got = at.attn_paged(q, k, v, own, lens, cu, n, prefix_table=table, prefix_len=total)
        kk, vv = torch.cat([k[4, :last], k[5]]), torch.cat([v[4, :last], v[5]])
        seen = last + torch.arange(page - n + 1, page + 1)
    else:
        lens = torch.tensor([total], dtype=torch.int32, device="cuda")
        got = at.attn_paged(q, k, v, table[None], lens, cu, n)
        kk, vv, seen = k[4, :last], v[4, :last], torch.arange(last - n + 1, last + 1)
    o, _, m = attend(q, kk, vv, seen, D ** -0.5)
    # sum |q k| / 8 is up to 60 + 20: 64 x 2^-24 of it, and 2^-23 of the exponent's argument, twice
    check(got, o, m, BF16, score_error=80 * 64 * 2.0 ** -24 + 2 * 115 * 2.0 ** -23 + 1e-4)
    hq.check_device_error()
