"""Split-fuse continuous batching over libhq.so (hq_batcher_*): the scheduling of hydrogen::SplitFuseBatcher
(batcher.hpp:98-199, split_fuse.cpp:70-193) with a step executor that runs real hq_gemm layers at the fused M
and, with a paged cache, the step's attention between them.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

from ._lib import HQ_ERR_INVALID_ARG, HQ_OK, HQError, check, lib

QUEUED, RUNNING_PREFILL, RUNNING_DECODE, COMPLETED = range(4)


class _Config(ctypes.Structure):
    _fields_ = [("max_prefill_chunk_tokens", ctypes.c_uint32), ("max_decode_streams", ctypes.c_uint32),
                ("max_batch_tokens", ctypes.c_uint32)]


class _Chunk(ctypes.Structure):
    _fields_ = [("request_id", ctypes.c_uint32), ("start_token", ctypes.c_uint32),
                ("num_tokens", ctypes.c_uint32), ("is_prefill", ctypes.c_int)]


class _Info(ctypes.Structure):
    _fields_ = [("num_decode_requests", ctypes.c_uint32), ("num_prefill_tokens", ctypes.c_uint32),
                ("total_batch_tokens", ctypes.c_uint32), ("assembly_overhead_us", ctypes.c_double)]


class _State(ctypes.Structure):
    _fields_ = [("prompt_tokens", ctypes.c_uint32), ("prefill_completed_tokens", ctypes.c_uint32),
                ("decode_tokens_generated", ctypes.c_uint32), ("max_decode_tokens", ctypes.c_uint32),
                ("status", ctypes.c_int)]


class LinearLayer(ctypes.Structure):
    """hq_linear_layer: one quantized linear layer (device pointers)."""
    _fields_ = [("W", ctypes.c_void_p), ("wfmt", ctypes.c_int), ("scales", ctypes.c_void_p),
                ("s_dtype", ctypes.c_int), ("bias", ctypes.c_void_p), ("K", ctypes.c_int), ("N", ctypes.c_int),
                ("group", ctypes.c_int)]


@dataclass
class BatchChunk:
    request_id: int
    start_token: int
    num_tokens: int
    is_prefill: bool


@dataclass
class FusedBatch:
    chunks: list
    num_decode_requests: int
    num_prefill_tokens: int
    total_batch_tokens: int
    assembly_overhead_us: float


@dataclass
class AttentionStep:
    """Where a fused batch's rows stand in the cache, as attention.attn_paged and kv_append take it (device tensors;
    sequence i is the i-th chunk that has rows)."""
    rows: int
    cu_q: object
    page_table: object
    kv_lens: object
    max_q_len: int
    max_kv_len: int
    prefix_table: object
    prefix_len: int
    stream: object = None     # the one that the plan was given
    planned_on: object = None  # that one, or the one that was current


class SplitFuseBatcher:
    """SplitFuseBatcher's scheduling surface: submit_request, assemble_step_batch, update_step_completion,
    has_active_work, num_active_requests, reset, and cancel_request; plus execute_step over real quantized layers.

    With a ``cache`` (attention.KVCache) the batcher keeps the requests' keys and values there: plan_attention makes
    room for a batch's rows, attend runs a layer's attention, update_step_completion frees what completed requests
    held.  ``prefix``: a sequence of the cache whose keys every request sees before its own.  All device work belongs
    on one stream, the current one or the one that plan_attention is given, and the cache is compacted between steps
    only."""

    def __init__(self, max_prefill_chunk_tokens=64, max_decode_streams=16, max_batch_tokens=512, *, cache=None,
                 prefix=None):
        self.cache, self.prefix = cache, prefix
        self._seqs = {}  # request -> (its sequence, keys that it began with)
        cfg = _Config(max_prefill_chunk_tokens, max_decode_streams, max_batch_tokens)
        self._h = lib().hq_batcher_create(ctypes.byref(cfg))
        if not self._h:
            raise MemoryError("hq_batcher_create")

    def close(self):
        if self._h:
            lib().hq_batcher_destroy(self._h)
            self._h = None
            for request in list(self._seqs):
                try:
                    self._release(request)
                except HQError:  # the cache is closed
                    pass

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def reset(self):
        lib().hq_batcher_reset(self._h)
        for request in list(self._seqs):
            self._release(request)

    def submit_request(self, prompt_tokens: int, max_decode_tokens: int, parent: int | None = None) -> int:
        """parent: an active request whose keys so far the new one continues; their pages are shared until either
        writes to them, and prompt_tokens counts the tokens after them."""
        if parent is not None and parent not in self._seqs:
            raise ValueError(f"request {parent} holds no keys")
        seq = self.cache.fork(self._seqs[parent][0]) if parent is not None else None
        try:
            request = int(lib().hq_batcher_submit(self._h, prompt_tokens, max_decode_tokens))
        except ctypes.ArgumentError:
            if seq is not None:
                self.cache.free(seq)
            raise
        if seq is not None:
            self._seqs[request] = seq, self.cache.pool.seq_len(seq)
        return request

    def cancel_request(self, request: int):
        """Gives an active request up, between two steps or where a step finds no pages: what it holds in the cache is
        freed, and batches are to be assembled anew."""
        status = lib().hq_batcher_cancel(self._h, request) if 0 < request < 2 ** 32 else HQ_ERR_INVALID_ARG
        if status != HQ_OK:
            raise HQError(status, f"no active request {request}")
        if request in self._seqs:
            self._release(request)

    def _release(self, request: int):
        self.cache.free(self._seqs.pop(request)[0])

    def assemble_step_batch(self) -> FusedBatch:
        cap = int(lib().hq_batcher_active_requests(self._h)) + 2
        buf = (_Chunk * cap)()
        info = _Info()
        n = lib().hq_batcher_assemble(self._h, buf, cap, ctypes.byref(info))
        if n < 0:
            raise RuntimeError("hq_batcher_assemble: chunk buffer too small")
        chunks = [BatchChunk(c.request_id, c.start_token, c.num_tokens, bool(c.is_prefill)) for c in buf[:n]]
        return FusedBatch(chunks, info.num_decode_requests, info.num_prefill_tokens, info.total_batch_tokens,
                          info.assembly_overhead_us)

    def update_step_completion(self, batch: FusedBatch):
        arr = (_Chunk * max(1, len(batch.chunks)))(
            *[_Chunk(c.request_id, c.start_token, c.num_tokens, int(c.is_prefill)) for c in batch.chunks])
        check(lib().hq_batcher_complete(self._h, arr, len(batch.chunks)))
        for c in batch.chunks:
            if c.request_id in self._seqs and self.request_state(c.request_id)["status"] == COMPLETED:
                self._release(c.request_id)

    def plan_attention(self, batch: FusedBatch, stream=None) -> AttentionStep:
        """Room in the cache for the batch's rows, for all or (HQ_ERR_OUT_OF_PAGES) for none, and their places.  To be
        called before the batch's attend; again for the same batch it gives the same.  The copies of pages that forks
        share run on ``stream``, which is attend's then, too."""
        import contextlib
        import numpy as np
        import torch
        cache = self.cache
        if cache is None:
            raise ValueError("the batcher has no cache")
        chunks = [c for c in batch.chunks if c.num_tokens]
        for c in chunks:
            if c.request_id not in self._seqs:
                if self.request_state(c.request_id)["status"] == COMPLETED:
                    raise ValueError(f"request {c.request_id} is not active")
                self._seqs[c.request_id] = cache.new_seq(), 0
        seqs = [self._seqs[c.request_id][0] for c in chunks]
        ends = [self._seqs[c.request_id][1] + c.start_token + c.num_tokens for c in chunks]
        cache.extend(seqs, [max(0, e - cache.pool.seq_len(s)) for s, e in zip(seqs, ends)], stream)
        table, _ = cache.pool.tables(seqs)
        prefix = cache.pool.seq_pages(self.prefix) if self.prefix is not None else np.empty(0, np.int32)
        n = len(seqs)
        counts = [c.num_tokens for c in chunks]
        host = np.concatenate([table.reshape(-1), prefix, np.array(ends, np.int32),
                               np.cumsum([0] + counts, dtype=np.int32)])
        on = stream
        if on is None and cache.k.is_cuda:
            on = torch.cuda.current_stream(cache.k.device)
        with torch.cuda.stream(stream) if stream is not None and cache.k.is_cuda else contextlib.nullcontext():
            dev = torch.from_numpy(host).to(cache.k.device)  # one copy for all four
        pages, pre, lens, cu = dev.split([table.size, prefix.size, n, n + 1])
        return AttentionStep(sum(counts), cu, pages.view(table.shape), lens, max(counts, default=0), max(ends, default=0), pre,
                             cache.pool.seq_len(self.prefix) if self.prefix is not None else 0, stream, on)

    def attend(self, step: AttentionStep, layer: int, q, k, v, *, scale=None, out=None, workspace=None, stream=None):
        """One layer's attention of a planned step: k and v [rows, Hkv, D] go into the layer's pages, then q
        [rows, Hq, D] attends to its sequences' keys.  Returns [rows, Hq, D].  On the stream that the plan was given,
        else on the current one; ``stream`` may name the plan's own, no other."""
        import torch

        from . import attention
        if stream is None:
            stream = step.stream
        elif step.planned_on is not None and stream.cuda_stream != step.planned_on.cuda_stream and \
                not (q.is_cuda and torch.cuda.is_current_stream_capturing()):  # a captured call runs where it is replayed
            raise ValueError("attend on another stream than plan_attention's, whose page copies it would not wait for")
        if q.shape[0] != step.rows or min(k.shape[0], v.shape[0]) < step.rows:
            raise ValueError(f"{q.shape[0]} rows for a step of {step.rows}, with {k.shape[0]} keys and {v.shape[0]} values")
        kp, vp = self.cache.k[layer], self.cache.v[layer]
        attention.kv_append(k, v, kp, vp, step.page_table, step.kv_lens, step.cu_q, stream=stream)
        return attention.attn_paged(q, kp, vp, step.page_table, step.kv_lens, step.cu_q, step.max_q_len,
                                    max_kv_len=step.max_kv_len, prefix_table=step.prefix_table,
                                    prefix_len=step.prefix_len, scale=scale, out=out, workspace=workspace, stream=stream)

    def has_active_work(self) -> bool:
        return bool(lib().hq_batcher_has_work(self._h))

    def num_active_requests(self) -> int:
        return int(lib().hq_batcher_active_requests(self._h))

    def request_state(self, request_id: int) -> dict:
        st = _State()
        check(lib().hq_batcher_request_state(self._h, request_id, ctypes.byref(st)))
        return {f: getattr(st, f) for f, _ in _State._fields_}

    def execute_step(self, rows: int, layers, act0, act1, a_dtype: int, workspace=None, stream=None):
        """Run `rows` rows of act0 through `layers` (LinearLayer list) with hq_gemm; returns the output buffer."""
        import torch
        arr = (LinearLayer * max(1, len(layers)))(*layers)
        s = stream if stream is not None else torch.cuda.current_stream()
        ws = ctypes.c_void_p(workspace.data_ptr()) if workspace is not None else None
        ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
        check(lib().hq_batcher_execute(self._h, rows, arr, len(layers), ctypes.c_void_p(act0.data_ptr()),
                                       ctypes.c_void_p(act1.data_ptr()), a_dtype, ws, ws_bytes,
                                       ctypes.c_void_p(s.cuda_stream)))
        return act1 if len(layers) % 2 else act0
