"""The operators together, as a server runs them: split-fuse batches through quantized QKV and output layers with the
paged attention between them, requests that share a prefix or fork, compactions; every step's attention against its
definition in 64 bits over plain lists of each request's keys."""
import random

import pytest
import torch

from attn_ref import attend, check
from nebula_b200 import hq
from nebula_b200.attention import KVCache, attn_prompt, kv_append
from nebula_b200.batcher import SplitFuseBatcher
from oracle import oracle as o

pytestmark = pytest.mark.gpu


def linear(K, N, seed, dtype):
    _, q, S = o.gen_int4_case(1, K, N, 128, seed=seed)
    return torch.from_numpy(o.pack_tile(q, 4)).cuda(), torch.from_numpy(S).cuda().to(dtype), N


@pytest.mark.parametrize("dtype,Hq,Hk,D,page,prefix_len", [(torch.float16, 8, 2, 64, 16, 0), (torch.bfloat16, 4, 4, 128, 64, 70),
                                                         (torch.bfloat16, 10, 2, 128, 16, 300)])
def test_batches_through_layers_and_cache(dtype, Hq, Hk, D, page, prefix_len):
    layers, hidden = 2, 512
    qkv = [linear(hidden, (Hq + 2 * Hk) * D, 10 + i, dtype) for i in range(layers)]
    proj = [linear(Hq * D, hidden, 20 + i, dtype) for i in range(layers)]
    cache = KVCache(layers, 1 + 2048 // page, page, Hk, D, dtype=dtype)
    num = cache.pool.free_pages
    gen, r = torch.Generator(device="cuda").manual_seed(3), random.Random(3)

    def gemm(x, layer):
        W, S, N = layer
        return hq.gemm(x, W, S, N=N, group=128)

    def heads(x, layer):
        y = gemm(x, qkv[layer]).view(x.shape[0], Hq + 2 * Hk, D)
        return y[:, :Hq], y[:, Hq: Hq + Hk], y[:, Hq + Hk:]

    def rms(x):  # keeps the rows at unit size, layer after layer
        return torch.nn.functional.rms_norm(x.float(), (hidden,)).to(dtype)

    pre, shared = [], None
    if prefix_len:  # its keys: one prompt through the layers
        shared = cache.new_seq()
        cache.extend([shared], [prefix_len])
        table, lens, _ = cache.tables([shared])
        x = torch.randn((prefix_len, hidden), generator=gen, device="cuda").to(dtype)
        cu = torch.tensor([0, prefix_len], dtype=torch.int32, device="cuda")
        for i in range(layers):
            q, k, v = heads(x, i)
            kv_append(k, v, cache.k[i], cache.v[i], table, lens, cu)
            got = attn_prompt(q, k, v, cu, prefix_len)
            ref, _, mag = attend(q, k, v, torch.arange(1, prefix_len + 1), D ** -0.5)
            check(got, ref, mag, dtype, 3e-4)
            pre.append((k, v))
            x = rms(gemm(got.reshape(prefix_len, Hq * D), proj[i]))
    b = SplitFuseBatcher(64, 16, 96, cache=cache, prefix=shared)
    plain = {}  # request -> per layer (k, v)
    none = [(torch.empty((0, Hk, D), dtype=dtype, device="cuda"),) * 2 for _ in range(layers)]
    for prompt in (1, 130, 17):
        plain[b.submit_request(prompt, 6)] = pre or none
    left, steps = 5, 0
    while b.has_active_work():
        if left and steps % 2:
            left -= 1
            parent = r.choice(sorted(b._seqs))
            plain[b.submit_request(r.choice([0, 3, 40]), 5, parent)] = plain[parent]
        if steps % 4 == 3:
            cache.compact()
        batch = b.assemble_step_batch()
        step = b.plan_attention(batch)
        chunks = [c for c in batch.chunks if c.num_tokens]
        x = torch.randn((step.rows, hidden), generator=gen, device="cuda").to(dtype)
        for i in range(layers if step.rows else 0):
            q, k, v = heads(x, i)
            got = b.attend(step, i, q, k, v)
            a = 0
            for c in chunks:
                n = c.num_tokens
                pk, pv = (torch.cat([old, new[a: a + n]]) for old, new in zip(plain[c.request_id][i], (k, v)))
                plain[c.request_id] = plain[c.request_id][:i] + [(pk, pv)] + plain[c.request_id][i + 1:]
                m = pk.shape[0]
                ref, _, mag = attend(q[a: a + n], pk, pv, torch.arange(m - n + 1, m + 1), D ** -0.5)
                check(got[a: a + n], ref, mag, dtype, 3e-4)  # the layers' outputs reach about 1.4 times N(0, 1)'s
                a += n
            x = rms(gemm(got.reshape(step.rows, Hq * D), proj[i]))
        b.update_step_completion(batch)
        steps += 1
    assert steps > 8 and left == 0
    if shared is not None:
        cache.free(shared)
    assert cache.pool.free_pages == num
    hq.check_device_error()
    b.close()


def test_a_step_without_rows():
    """A request with no prompt is a chunk of no rows: nothing runs, and its decode steps follow."""
    cache = KVCache(1, 4, 16, 2, 64, dtype=torch.float16)
    b = SplitFuseBatcher(cache=cache)
    b.submit_request(0, 1)
    for rows in (0, 1):
        batch = b.assemble_step_batch()
        step = b.plan_attention(batch)
        q, k = torch.randn((rows, 4, 64), device="cuda").half(), torch.randn((rows, 2, 64), device="cuda").half()
        got = b.attend(step, 0, q, k, k)
        assert got.shape == q.shape and torch.equal(got, k.repeat_interleave(2, 1))  # one key: its value
        b.update_step_completion(batch)
    assert not b.has_active_work() and cache.pool.free_pages == 4
    hq.check_device_error()
    b.close()
