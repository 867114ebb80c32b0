"""A batcher whose device work is on a stream of its own."""
import pytest
import torch

from attn_ref import attend, check
from nebula_b200 import hq
from nebula_b200.attention import KVCache
from nebula_b200.batcher import SplitFuseBatcher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("given", [True, False])
def test_forks_on_a_side_stream(given):
    """Plans and layers on a stream that is not the current one, or under it; forks that copy a partly filled page in
    every step, while the current stream is busy."""
    Hq, Hk, D, layers, page = 4, 2, 64, 2, 256
    cache = KVCache(layers, 40, page, Hk, D, dtype=torch.float16)
    b = SplitFuseBatcher(64, 16, 96, cache=cache)
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda n, h: torch.randn((n, h, D), generator=g, device="cuda", dtype=torch.float16)  # noqa: E731
    plain = {b.submit_request(60, 20): [(rnd(0, Hk), rnd(0, Hk))] * layers}
    busy = torch.zeros(1 << 28, device="cuda")
    side = torch.cuda.Stream()
    for i in range(12):
        if i in (2, 4, 5, 8):
            parent = min(b._seqs)
            plain[b.submit_request(1 + i, 20, parent)] = list(plain[parent])
        batch = b.assemble_step_batch()
        rows = batch.total_batch_tokens
        data = [(rnd(rows, Hq), rnd(rows, Hk), rnd(rows, Hk)) for _ in range(layers)]
        torch.cuda.synchronize()
        for _ in range(4):
            busy.add_(1.0)
        if given:
            step = b.plan_attention(batch, stream=side)
            got = [b.attend(step, j, *data[j], stream=side if j else None) for j in range(layers)]
        else:
            with torch.cuda.stream(side):
                step = b.plan_attention(batch)
                got = [b.attend(step, j, *data[j], stream=side if j else None) for j in range(layers)]
            with pytest.raises(ValueError, match="another stream"):
                b.attend(step, 0, *data[0], stream=torch.cuda.current_stream())
        side.synchronize()
        for j, (q, k, v) in enumerate(data):
            a = 0
            for c in batch.chunks:
                n = c.num_tokens
                pk, pv = (torch.cat([old, new[a: a + n]]) for old, new in zip(plain[c.request_id][j], (k, v)))
                plain[c.request_id] = plain[c.request_id][:j] + [(pk, pv)] + plain[c.request_id][j + 1:]
                m = pk.shape[0]
                ref, _, mag = attend(q[a: a + n], pk, pv, torch.arange(m - n + 1, m + 1), D ** -0.5)
                check(got[j][a: a + n], ref, mag, torch.float16)
                a += n
        b.update_step_completion(batch)
    hq.check_device_error()
    b.close()


@pytest.mark.parametrize("named", [False, True])
def test_a_planned_step_in_a_captured_call(named):
    """Planned on the current stream, captured on the capture's own."""
    cache = KVCache(1, 8, 16, 2, 64, dtype=torch.float16)
    b = SplitFuseBatcher(cache=cache)
    b.submit_request(30, 4)
    step = b.plan_attention(b.assemble_step_batch())
    q, k, v = (torch.randn((30, h, 64), device="cuda").half() for h in (4, 2, 2))
    out = torch.zeros_like(q)
    b.attend(step, 0, q, k, v, out=out)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        b.attend(step, 0, q, k, v, out=out, stream=s if named else None)
    for t in (q, k, v):
        t.normal_()
    graph.replay()
    ref, _, mag = attend(q, k, v, torch.arange(1, 31), 64 ** -0.5)
    check(out, ref, mag, torch.float16)
    hq.check_device_error()
    b.close()
