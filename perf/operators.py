"""The attention and key/value-cache operators: what is timed, their plain forms, and their definition in 64 bits.

Five operators, as a serving step of a decoder uses them:
  prompt   causal attention of whole prompts, packed one behind the other, grouped heads
  step     attention of a split-fuse step over a paged cache (one row a stream, and prompt chunks)
  prefix   the same for a batch whose sequences share a long prefix, read once for all of them
  append   the step's new keys and values written into the pages
  pages    pages copied in place (copy-on-write after a fork, the moves of a compaction), all layers at once

Head layouts are those of the 27B layer this framework is sized for (QKV 5120 x 7168: 40 query and 8 key/value heads
of 128), its shards over 4 and 8 GPUs, and plain multi-head and single-key-head layouts with heads of 64.
"""
import math
import random

import numpy as np
import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
LAYOUTS = [(40, 8, 128), (10, 2, 128), (5, 1, 128), (32, 4, 128), (16, 16, 64), (8, 1, 64)]


def listed():
    return [
        # three short questions on one of four tensor-parallel shards: the smallest call, its latency counts
        dict(name="prompt_short", op="prompt", type="f16", heads=10, kv_heads=2, dim=128, sequences=3, longest=61),
        # a dozen prompts of different lengths in one batch, plain multi-head layout
        dict(name="prompt_ragged", op="prompt", type="f16", heads=16, kv_heads=16, dim=64, sequences=12, longest=1500),
        # one long document, whole model on one GPU
        dict(name="prompt_long", op="prompt", type="bf16", heads=40, kv_heads=8, dim=128, sequences=1, longest=8192),
        # one chat stream, one token
        dict(name="step_single", op="step", type="bf16", heads=40, kv_heads=8, dim=128, sequences=1, longest=777, page=16,
             chunk=0),
        # the batcher's own step: 16 streams and a 64-token chunk of a 1500-token observation
        dict(name="step_split_fuse", op="step", type="f16", heads=40, kv_heads=8, dim=128, sequences=17, longest=1500, page=16,
             chunk=64),
        # many long streams, one token each
        dict(name="step_long", op="step", type="bf16", heads=40, kv_heads=8, dim=128, sequences=64, longest=16001, page=32,
             chunk=0),
        # a few answers sampled behind one system prompt, one of eight shards
        dict(name="prefix_short", op="prefix", type="f16", heads=5, kv_heads=1, dim=128, sequences=8, longest=99, page=16,
             prefix=1024),
        # a batch of questions on one long document
        dict(name="prefix_long", op="prefix", type="bf16", heads=40, kv_heads=8, dim=128, sequences=64, longest=500, page=64,
             prefix=32001),
        # a step's rows: 16 streams and a chunk
        dict(name="append_step", op="append", type="f16", heads=40, kv_heads=8, dim=128, sequences=17, longest=1500, page=16,
             chunk=64),
        # whole prompts written after their prefill
        dict(name="append_prompts", op="append", type="bf16", heads=40, kv_heads=8, dim=128, sequences=8, longest=4001,
             page=32, chunk=4001),
        # eight forks of a stream write on: the last page of each is copied, in four layers
        dict(name="pages_fork", op="pages", type="f16", heads=40, kv_heads=8, dim=128, layers=4, page=16, pool=256, moves=8),
        # a compaction of a fragmented pool
        dict(name="pages_compact", op="pages", type="bf16", heads=40, kv_heads=8, dim=128, layers=16, page=32, pool=2048,
             moves=801),
    ]


def draw(rng):
    def log(a, b):
        return min(b, max(a, round(math.exp(rng.uniform(math.log(a), math.log(b))))))

    heads, kv_heads, dim = rng.choice(LAYOUTS)
    c = dict(op=rng.choice(["prompt", "step", "step", "prefix", "append", "pages"]), type=rng.choice(["f16", "bf16"]),
             heads=heads, kv_heads=kv_heads, dim=dim)
    if c["op"] == "prompt":
        c["sequences"] = log(1, 24)
        c["longest"] = log(1, int(8000 / math.sqrt(c["sequences"])))
        return c
    c["page"] = rng.choice([16, 32, 64, 128])
    if c["op"] == "pages":
        c["layers"] = log(1, 16)
        c["pool"] = log(64, min(2048, 16 * 2048 * 32 // (c["layers"] * c["page"])))
        c["moves"] = log(1, int(0.39 * c["pool"]))
        return c
    c["sequences"] = log(1, 64)
    if c["op"] == "prefix":
        c["longest"], c["prefix"] = log(1, 600), log(40, 32000)
        return c
    c["longest"] = log(1, int(16000 * min(1.0, 16 / c["sequences"])))
    if c["op"] == "step":
        room = int(2e9 / (c["sequences"] * c["longest"] * heads))  # the plain form pads every sequence to the chunk
        c["chunk"] = rng.choice([0, 0, min(c["longest"], room, log(2, 500))])
    else:
        c["chunk"] = rng.choice([0, min(c["longest"], log(2, 4000))])
    return c


def _lengths(c):
    """Ragged lengths, the same for every seed: the longest first, the others spread between a tenth of it and all of it."""
    r = random.Random(c["longest"] * 131 + c["sequences"])
    low = max(1, c["longest"] // 10)
    lens = [c["longest"]] + [r.randint(low, c["longest"]) for _ in range(c["sequences"] - 1)]
    if c["op"] == "prompt" or c.get("chunk", 0) == 0 or c["sequences"] == 1:
        return lens
    return lens[1:] + lens[:1]  # the chunk's sequence comes last, as in a split-fuse step


def _queries(c):
    """New tokens of each sequence. An append whose chunk is as long as the longest writes every sequence whole."""
    lens = _lengths(c)
    if c["op"] == "prompt":
        return lens
    if c.get("chunk", 0) == 0:
        return [1] * len(lens)
    if c["op"] == "append" and c["chunk"] >= c["longest"]:
        return lens
    return [1] * (len(lens) - 1) + [c["chunk"]]


def _cu(n):
    return [0] + list(np.cumsum(n))


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, D, H, Hk = DT[c["type"]], c["dim"], c["heads"], c["kv_heads"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dt)

    s = dict(c=c)
    if c["op"] == "pages":
        s["k"], s["v"] = (randn(c["layers"], c["pool"], c["page"], Hk, D) for _ in range(2))
        order = np.random.RandomState(seed % (1 << 31)).permutation(c["pool"])[: 2 * c["moves"]].astype(np.int32)
        s["src"], s["dst"] = order[: c["moves"]].copy(), order[c["moves"]:].copy()
        return s
    q_lens = _queries(c)
    T = sum(q_lens)
    # rows as the QKV layer leaves them: queries, keys and values of a token side by side
    qkv = randn(T, (H + 2 * Hk) * D)
    s["q"] = qkv[:, : H * D].view(T, H, D)
    s["new_k"] = qkv[:, H * D: (H + Hk) * D].view(T, Hk, D)
    s["new_v"] = qkv[:, (H + Hk) * D:].view(T, Hk, D)
    s["cu"] = torch.tensor(_cu(q_lens), dtype=torch.int32, device="cuda")
    s["max_q"] = max(q_lens)
    if c["op"] == "prompt":
        return s
    P = c["page"]
    lens = _lengths(c)
    used = [-(-n // P) for n in lens]
    prefix_pages = -(-c.get("prefix", 0) // P)
    pool = sum(used) + prefix_pages + 3
    s["k"], s["v"] = randn(pool, P, Hk, D), randn(pool, P, Hk, D)
    perm = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(used)), dtype=torch.int32, device="cuda")
    have = torch.arange(max(used), device="cuda")[None] < torch.tensor(used, device="cuda")[:, None]
    table[have] = perm[: sum(used)]
    s["table"] = table
    s["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["max_kv"] = max(lens)
    if c["op"] == "prefix":
        s["prefix_table"] = perm[sum(used): sum(used) + prefix_pages].clone()
        s["prefix_len"] = c["prefix"]
    return s


# ------------------------------------------------------------------ plain forms


def _padded(x, cu, width):
    """[T, ...] packed rows -> [B, width, ...] in 32 bits, and which of them exist."""
    at = torch.arange(width, device=x.device)
    have = at[None] < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + at[None]).clamp(max=x.shape[0] - 1).long()
    return x[rows].float(), have


def _softmax(scores, seen):
    """Softmax over the last dimension where `seen`; rows that see nothing give zeros."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_prompt(s):
    c = s["c"]
    G, scale = c["heads"] // c["kv_heads"], 1.0 / math.sqrt(c["dim"])
    q, have = _padded(s["q"], s["cu"], s["max_q"])
    k, _ = _padded(s["new_k"], s["cu"], s["max_q"])
    v, _ = _padded(s["new_v"], s["cu"], s["max_q"])
    B, L = have.shape
    q = q.view(B, L, c["kv_heads"], G, c["dim"]).permute(0, 2, 3, 1, 4).reshape(B, c["kv_heads"], G * L, c["dim"])
    at = torch.arange(L, device=q.device)
    seen = (at[None, :] <= at[:, None]).repeat(G, 1)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * scale
    p = _softmax(scores, seen & have[:, None, None, :])
    o = torch.matmul(p, v.permute(0, 2, 1, 3)).view(B, c["kv_heads"], G, L, c["dim"])
    return o.permute(0, 3, 1, 2, 4).reshape(B, L, c["heads"], c["dim"])[have].to(s["q"].dtype)


def _plain_paged(s):
    c = s["c"]
    G, scale = c["heads"] // c["kv_heads"], 1.0 / math.sqrt(c["dim"])
    q, have = _padded(s["q"], s["cu"], s["max_q"])
    B, L = have.shape
    Hk, D, P = c["kv_heads"], c["dim"], c["page"]
    q = q.view(B, L, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * L, D)
    k, v = (s[n][s["table"].long()].flatten(1, 2).float() for n in "kv")  # [B, S, Hk, D]
    at = torch.arange(k.shape[1], device=q.device)
    last = s["kv_lens"][:, None] - (s["cu"][1:] - s["cu"][:-1])[:, None] + torch.arange(L, device=q.device)[None]
    seen = (at[None, None] <= last[..., None]) & (at[None, None] < s["kv_lens"][:, None, None])
    seen = seen[:, None, None].expand(B, 1, G, L, -1).reshape(B, 1, G * L, -1)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * scale
    if c["op"] == "prefix":
        pk, pv = (s[n][s["prefix_table"].long()].flatten(0, 1)[: s["prefix_len"]].float() for n in "kv")  # [S, Hk, D]
        first = torch.matmul(q, pk.permute(1, 2, 0)) * scale
        scores = torch.cat([first, scores], -1)
        seen = torch.cat([torch.ones_like(first[:, :1], dtype=torch.bool), seen], -1)
    p = _softmax(scores, seen)
    if c["op"] == "prefix":
        n = s["prefix_len"]
        o = torch.matmul(p[..., :n], pv.permute(1, 0, 2)) + torch.matmul(p[..., n:], v.permute(0, 2, 1, 3))
    else:
        o = torch.matmul(p, v.permute(0, 2, 1, 3))
    o = o.view(B, Hk, G, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, c["heads"], D)
    return o[have].to(s["q"].dtype)


def _plain_append(s):
    P = s["c"]["page"]
    cu = s["cu"].long()
    T = s["new_k"].shape[0]
    row = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu, row, right=True) - 1
    pos = s["kv_lens"][b] - (cu[b + 1] - row)
    page = s["table"][b, pos // P].long()
    s["k"][page, pos % P] = s["new_k"]
    s["v"][page, pos % P] = s["new_v"]
    return s["k"], s["v"]


def _plain_pages(s):
    src, dst = (torch.from_numpy(s[n]).cuda().long() for n in ("src", "dst"))
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["k"], s["v"]


def run(s):
    op = s["c"]["op"]
    if own:
        from nebula_b200 import attention as at
        if op == "prompt":
            return at.attn_prompt(s["q"], s["new_k"], s["new_v"], s["cu"], s["max_q"])
        if op == "step":
            return at.attn_paged(s["q"], s["k"], s["v"], s["table"], s["kv_lens"], s["cu"], s["max_q"], max_kv_len=s["max_kv"])
        if op == "prefix":
            return at.attn_paged(s["q"], s["k"], s["v"], s["table"], s["kv_lens"], s["cu"], s["max_q"], max_kv_len=s["max_kv"],
                                 prefix_table=s["prefix_table"], prefix_len=s["prefix_len"])
        if op == "append":
            at.kv_append(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["kv_lens"], s["cu"])
            return s["k"], s["v"]
        at.kv_copy_pages([s["k"], s["v"]], s["src"], s["dst"])
        return s["k"], s["v"]
    if op == "prompt":
        return _plain_prompt(s)
    if op in ("step", "prefix"):
        return _plain_paged(s)
    return _plain_append(s) if op == "append" else _plain_pages(s)


def work(case):
    c = case
    row = c["kv_heads"] * c["dim"] * 2  # bytes of one token's keys (or values)
    if c["op"] == "pages":
        return {"bytes": 2 * 2 * c["layers"] * c["moves"] * c["page"] * row, "flops": 0}
    q_lens = _queries(c)
    T = sum(q_lens)
    if c["op"] == "append":
        return {"bytes": 2 * 2 * T * row, "flops": 0}
    q_bytes = 2 * T * c["heads"] * c["dim"] * 2  # queries in, outputs out
    if c["op"] == "prompt":
        pairs = sum(n * (n + 1) // 2 for n in q_lens)
        return {"bytes": q_bytes + 2 * T * row, "flops": 4 * pairs * c["heads"] * c["dim"]}
    lens = _lengths(c)
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q_lens, lens)) + T * c.get("prefix", 0)
    return {"bytes": q_bytes + 2 * (sum(lens) + c.get("prefix", 0)) * row, "flops": 4 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------------ the definition, in 64 bits


def _attend(q, k, v, first, scale):
    """One sequence and key head: q [n, G, D], k and v [m, D]; query i sees the keys at places <= first + i."""
    n, G, D = q.shape
    out = torch.empty(n, G, v.shape[1], dtype=torch.float64, device=q.device)
    for a in range(0, n, 1024):
        b = min(n, a + 1024)
        m = min(k.shape[0], first + b)
        w = torch.einsum("ngd,md->ngm", q[a:b].double(), k[:m].double()) * scale
        late = torch.arange(m, device=q.device)[None, :] > (first + torch.arange(a, b, device=q.device))[:, None]
        w = torch.softmax(w.masked_fill(late[:, None, :], -math.inf), -1)
        out[a:b] = torch.einsum("ngm,md->ngd", w, v[:m].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["op"] == "pages":
        if s["k"].numel() > (1 << 30):
            return None
        got = [s["k"].double(), s["v"].double()]
        for t in got:
            old = t.clone()
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                t[:, b].copy_(old[:, a])
        return tuple(got)
    cu = s["cu"].tolist()
    if c["op"] == "append":
        got = [s["k"].double(), s["v"].double()]
        for b, end in enumerate(s["kv_lens"].tolist()):
            pages = s["table"][b].tolist()
            place = end - (cu[b + 1] - cu[b])
            row = cu[b]
            while row < cu[b + 1]:  # a run of rows within one page
                n = min(c["page"] - place % c["page"], cu[b + 1] - row)
                for t, new in zip(got, (s["new_k"], s["new_v"])):
                    t[pages[place // c["page"]], place % c["page"]: place % c["page"] + n] = new[row: row + n].double()
                row, place = row + n, place + n
        return tuple(got)
    G, scale = c["heads"] // c["kv_heads"], c["dim"] ** -0.5
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(len(cu) - 1):
        rows = slice(cu[b], cu[b + 1])
        n = cu[b + 1] - cu[b]
        for h in range(c["kv_heads"]):
            if c["op"] == "prompt":
                k, v, first = s["new_k"][rows, h], s["new_v"][rows, h], 0
            else:
                m = int(s["kv_lens"][b])
                pages = s["table"][b, : -(-m // c["page"])].long()
                k, v = (s[name][pages, :, h].reshape(-1, c["dim"])[:m] for name in "kv")
                first = m - n
                if c["op"] == "prefix":
                    pages = s["prefix_table"].long()
                    before = [s[name][pages, :, h].reshape(-1, c["dim"])[: s["prefix_len"]] for name in "kv"]
                    k, v = torch.cat([before[0], k]), torch.cat([before[1], v])
                    first += s["prefix_len"]
            out[rows, h * G: (h + 1) * G] = _attend(s["q"][rows, h * G: (h + 1) * G], k, v, first, scale)
    return out
