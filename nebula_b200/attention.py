"""Attention and its paged key/value cache (torch tensors in, libhq.so underneath).

  * ``attn_prompt`` -- causal (or full) attention within packed prompts;
  * ``attn_paged``  -- a split-fuse step's rows over a paged cache, decode rows and prompt chunks alike, with an
    optional prefix that all sequences share and that is read once (the reference's decoder attention,
    hydrogen/src/model/native_decoder.cu:263, and hydrogen/src/attention/cascade_attention.cu);
  * ``kv_append``   -- the step's new keys and values into their pages;
  * ``kv_copy_pages`` -- pages over other pages, all layers in one call;
  * ``PagePool`` / ``KVCache`` -- which pages belong to which sequence (fork, extend, free, compact), without and
    with the cache's memory.

q, k, v and out are [tokens, heads, head_dim] float16 or bfloat16 (slices of the QKV layer's output do: only
head_dim is contiguous); a cache is [num_pages, page_size, kv_heads, head_dim], any order of the outer strides.
Row offsets, lengths and page tables are int32 device tensors, read when the kernels run.  All device work runs on
``stream`` or the caller's current torch stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _lib
from ._lib import HQ_BF16, HQ_F16, HQError, check, lib

__all__ = ["attn_prompt", "attn_paged", "kv_append", "kv_copy_pages", "PagePool", "KVCache"]

_ref = ctypes.byref
_DT = {torch.float16: HQ_F16, torch.bfloat16: HQ_BF16}


class _Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("stride_token", ctypes.c_int64), ("stride_head", ctypes.c_int64)]


class _Pages(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("stride_page", ctypes.c_int64), ("stride_token", ctypes.c_int64),
                ("stride_head", ctypes.c_int64)]


class _Shape(ctypes.Structure):
    _fields_ = [("n_tokens", ctypes.c_int), ("n_seqs", ctypes.c_int), ("max_q_len", ctypes.c_int),
                ("n_heads", ctypes.c_int), ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("dtype", ctypes.c_int), ("scale", ctypes.c_float)]


class _View(ctypes.Structure):
    _fields_ = [("k", _Pages), ("v", _Pages), ("num_pages", ctypes.c_int), ("page_size", ctypes.c_int),
                ("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("max_pages", ctypes.c_int),
                ("kv_lens", ctypes.c_void_p)]


class _Move(ctypes.Structure):
    _fields_ = [("src", ctypes.c_int32), ("dst", ctypes.c_int32)]


def _bad(msg: str):
    raise HQError(_lib.HQ_ERR_INVALID_ARG, msg)


def _rows(t: torch.Tensor, name: str, like: torch.Tensor, heads: int) -> _Rows:
    if t.dim() != 3 or t.shape[0] != like.shape[0] or t.shape[1] != heads or t.shape[2] != like.shape[2]:
        _bad(f"{name} must be [{like.shape[0]}, {heads}, {like.shape[2]}], got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        _bad(f"{name}: {t.dtype} on {t.device} beside {like.dtype} on {like.device}")
    st, sh, sd = t.stride()
    if sd != 1:
        _bad(f"{name}: head_dim must be contiguous")
    return _Rows(t.data_ptr(), st, sh)


def _pages(t: torch.Tensor, name: str, like: torch.Tensor) -> _Pages:
    if t.dim() != 4 or t.shape[3] != like.shape[2]:
        _bad(f"{name} must be [num_pages, page_size, kv_heads, {like.shape[2]}], got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        _bad(f"{name}: {t.dtype} on {t.device} beside {like.dtype} on {like.device}")
    sp, st, sh, sd = t.stride()
    if sd != 1:
        _bad(f"{name}: head_dim must be contiguous")
    return _Pages(t.data_ptr(), sp, st, sh)


def _index(t: torch.Tensor | None, name: str, shape: tuple, like: torch.Tensor):
    """Device address of an int32 index tensor (None: null)."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.device != like.device or tuple(t.shape) != shape:
        _bad(f"{name} must be int32 {list(shape)} on {like.device}, got {t.dtype} {list(t.shape)} on {t.device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        _bad(f"{name} must be contiguous")
    return t.data_ptr()


def _view(k_pages, v_pages, page_table, kv_lens, like) -> tuple[_View, int]:
    if k_pages.shape != v_pages.shape:
        _bad(f"key pages {tuple(k_pages.shape)} and value pages {tuple(v_pages.shape)} differ")
    k, v = _pages(k_pages, "k_pages", like), _pages(v_pages, "v_pages", like)
    if page_table.dim() != 2:
        _bad("page_table must be [sequences, pages]")
    n = page_table.shape[0]
    table = _index(page_table, "page_table", (n, page_table.shape[1]), like)
    return _View(k, v, k_pages.shape[0], k_pages.shape[1], table, page_table.stride(0), page_table.shape[1],
                 _index(kv_lens, "kv_lens", (n,), like)), n


def _dtype(q: torch.Tensor) -> int:
    dt = _DT.get(q.dtype)
    if dt is None:
        _bad(f"unsupported dtype {q.dtype}")
    if q.device.type != "cuda":
        _bad(f"tensors must be on a CUDA device, got {q.device}")
    return dt


class _On:
    """The device and stream of a call: makes `device` current where it is not, allocates on the launch stream."""
    __slots__ = ("ptr", "ctx")

    def __init__(self, device: torch.device, stream):
        self.ctx = None
        if stream is not None:
            if stream.device != device:
                _bad(f"a stream of {stream.device} for tensors on {device}")
            self.ctx = torch.cuda.stream(stream)
        elif device.index is not None and device.index != torch.cuda.current_device():
            self.ctx = torch.cuda.device(device)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()
        self.ptr = torch.cuda.current_stream().cuda_stream
        return self.ptr

    def __exit__(self, *e):
        if self.ctx is not None:
            self.ctx.__exit__(*e)


def _outputs(q, out, lse, heads):
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse_p = None
    if lse is not None:
        if lse.dtype != torch.float32 or tuple(lse.shape) != (q.shape[0], heads) or not lse.is_contiguous() or \
                lse.device != q.device:
            _bad(f"lse must be contiguous float32 [{q.shape[0]}, {heads}] on {q.device}")
        lse_p = lse.data_ptr()
    return out, _rows(out, "out", q, heads), lse_p


def _workspace(need: int, workspace, device):
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device) if need else None
    if workspace.device != device or not workspace.is_contiguous():
        _bad(f"workspace must be contiguous on {device}")
    return workspace


def _ws_args(ws):
    return (None, 0) if ws is None else (ws.data_ptr(), ws.numel() * ws.element_size())


def attn_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int, *,
                causal: bool = True, scale: float | None = None, out: torch.Tensor | None = None,
                lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention within packed sequences: q [T, Hq, D], k and v [T, Hkv, D]; sequence s is the rows
    cu_seqlens[s] .. cu_seqlens[s+1]-1, at most max_seqlen of them.  Rows behind the last sequence keep what `out`
    holds.  lse: optional [T, Hq] float32 output (ln of the softmax denominator)."""
    dt = _dtype(q)
    if q.dim() != 3 or k.dim() != 3 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        _bad("q, k, v must be [tokens, heads, head_dim], cu_seqlens [sequences + 1]")
    T, Hq, D = q.shape
    Hk, B = k.shape[1], cu_seqlens.numel() - 1
    rk, rv, rq = _rows(k, "k", q, Hk), _rows(v, "v", q, Hk), _rows(q, "q", q, Hq)
    cu = _index(cu_seqlens, "cu_seqlens", (B + 1,), q)
    sh = _Shape(T, B, max_seqlen, Hq, Hk, D, dt, 1.0 / math.sqrt(D) if scale is None else scale)
    L = lib()
    with _On(q.device, stream) as s:
        out, ro, lse_p = _outputs(q, out, lse, Hq)
        ws = _workspace(L.hq_attn_prompt_workspace_size(_ref(sh)), workspace, q.device)
        check(L.hq_attn_prompt(_ref(sh), _ref(rq), _ref(rk), _ref(rv), cu, int(causal), _ref(ro), lse_p, *_ws_args(ws), s))
    return out


def attn_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
               kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, max_q_len: int = 1, *,
               max_kv_len: int | None = None, prefix_table: torch.Tensor | None = None, prefix_len: int = 0,
               scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention of a step's rows over a paged cache: q [T, Hq, D]; sequence s has the rows cu_q[s] .. cu_q[s+1]-1
    (cu_q None: row s alone), at most max_q_len, and kv_lens[s] keys, its rows' own last (kv_append writes them
    first).  Row i of n sees keys 0 .. kv_lens[s] - n + i, after the prefix_len keys of the pages prefix_table that
    every sequence shares.  max_kv_len: a bound of kv_lens that sizes the launch."""
    dt = _dtype(q)
    if q.dim() != 3:
        _bad("q must be [tokens, heads, head_dim]")
    T, Hq, D = q.shape
    view, B = _view(k_pages, v_pages, page_table, kv_lens, q)
    Hk = k_pages.shape[2]
    rq = _rows(q, "q", q, Hq)
    cu = _index(cu_q, "cu_q", (B + 1,), q)
    if max_kv_len is None:
        max_kv_len = view.max_pages * view.page_size
    pt = None
    if prefix_len:
        if prefix_table is None:
            _bad("prefix_len without prefix_table")
        pt = _index(prefix_table, "prefix_table", tuple(prefix_table.shape), q)
        if prefix_table.dim() != 1 or prefix_table.shape[0] * view.page_size < prefix_len:
            _bad(f"prefix_table {list(prefix_table.shape)} does not hold {prefix_len} keys")
    sh = _Shape(T, B, max_q_len, Hq, Hk, D, dt, 1.0 / math.sqrt(D) if scale is None else scale)
    L = lib()
    with _On(q.device, stream) as s:
        out, ro, lse_p = _outputs(q, out, lse, Hq)
        ws = _workspace(L.hq_attn_paged_workspace_size(_ref(sh), max_kv_len, prefix_len), workspace, q.device)
        check(L.hq_attn_paged(_ref(sh), _ref(rq), _ref(view), cu, max_kv_len, pt, prefix_len, _ref(ro), lse_p,
                              *_ws_args(ws), s))
    return out


def kv_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              page_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, *,
              stream=None) -> None:
    """Writes the rows of k and v [T, Hkv, D] into their pages: row i of the n rows of sequence s becomes its key
    kv_lens[s] - n + i."""
    dt = _dtype(k)
    if k.dim() != 3:
        _bad("k and v must be [tokens, kv_heads, head_dim]")
    T, Hk, D = k.shape
    view, B = _view(k_pages, v_pages, page_table, kv_lens, k)
    if k_pages.shape[2] != Hk:
        _bad(f"{Hk} heads into pages of {k_pages.shape[2]}")
    rk, rv = _rows(k, "k", k, Hk), _rows(v, "v", k, Hk)
    cu = _index(cu_q, "cu_q", (B + 1,), k)
    with _On(k.device, stream) as s:
        sh = _Shape(T, B, T, Hk, Hk, D, dt, 1.0)
        check(lib().hq_kv_append(_ref(sh), _ref(rk), _ref(rv), _ref(view), cu, s))


def _moves(src, dst):
    n = len(src)
    if len(dst) != n:
        _bad(f"{n} source pages and {len(dst)} destinations")
    both = np.empty((n, 2), np.int32)
    both[:, 0], both[:, 1] = src, dst
    return both, n


def kv_copy_pages(pools, src, dst, *, stream=None) -> None:
    """Copies page src[i] over page dst[i] (host integers) in every pool: tensors [num_pages, ...] of four
    dimensions, or [layers, num_pages, ...] of five, all of one geometry, a page being one block of memory.  A page
    may be copied to several places; one that is written twice, or read and written, is refused."""
    both, n = _moves(src, dst)
    bases, geometry = [], None
    for t in pools:
        if t.device.type != "cuda" or t.device != pools[0].device:
            _bad("pools must be on one CUDA device")
        if t.dim() not in (4, 5):
            _bad(f"a pool has 4 or 5 dimensions, got {tuple(t.shape)}")
        pages = t.dim() - 4
        size = t.element_size()
        inner = t[0, 0] if pages else t[0]
        # one block: the strides of the inner dimensions, ascending, are the running product of their sizes
        run = 1
        for st, n_ in sorted((st, n_) for st, n_ in zip(inner.stride(), inner.shape) if n_ > 1):
            if st != run:
                _bad(f"a page must be one block of memory, got strides {inner.stride()}")
            run *= n_
        g = (t.shape[pages], t.stride(pages) * size, run * size)
        if geometry not in (None, g):
            _bad("pools of different geometry")
        geometry = g
        if pages:
            step = t.stride(0) * size
            bases += [t.data_ptr() + i * step for i in range(t.shape[0])]
        else:
            bases.append(t.data_ptr())
    if not bases:
        return
    with _On(pools[0].device, stream) as s:
        check(lib().hq_kv_copy_pages((ctypes.c_void_p * len(bases))(*bases), len(bases), geometry[1], geometry[2],
                                     geometry[0], both.ctypes.data, n, s))


class PagePool:
    """Pages of a cache by sequence: reference counts and page lists on the host (hq_kv_pool_*)."""

    def __init__(self, num_pages: int, page_size: int):
        self._h = lib().hq_kv_pool_create(num_pages, page_size)
        if not self._h:
            _bad(f"no pool of {num_pages} pages of {page_size} (a power of two from 16 to 256)")
        self.num_pages, self.page_size = num_pages, page_size

    def close(self):
        if getattr(self, "_h", None):
            lib().hq_kv_pool_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def free_pages(self) -> int:
        return int(lib().hq_kv_pool_free_pages(self._h))

    def new_seq(self) -> int:
        s = int(lib().hq_kv_pool_new_seq(self._h))
        if s < 0:
            raise MemoryError("hq_kv_pool_new_seq")
        return s

    def fork(self, seq: int) -> int:
        """A sequence with the same keys; pages are shared until one of the two is extended."""
        s = int(lib().hq_kv_pool_fork(self._h, seq))
        if s < 0:
            _bad(f"no sequence {seq}")
        return s

    def extend(self, seq: int, n_tokens: int) -> list[tuple[int, int]]:
        """Room for n_tokens more keys; returns the page copies, (source, destination), to make first."""
        mv, n = _Move(), ctypes.c_int(0)
        status = lib().hq_kv_pool_extend(self._h, seq, n_tokens, ctypes.byref(mv), ctypes.byref(n))
        if status != _lib.HQ_OK:
            raise HQError(status, f"sequence {seq} by {n_tokens} keys, {self.free_pages} pages free")
        return [(mv.src, mv.dst)] if n.value else []

    def free(self, seq: int) -> None:
        status = lib().hq_kv_pool_free(self._h, seq)
        if status != _lib.HQ_OK:
            raise HQError(status, f"no sequence {seq}")

    def seq_len(self, seq: int) -> int:
        n = int(lib().hq_kv_pool_seq_len(self._h, seq))
        if n < 0:
            _bad(f"no sequence {seq}")
        return n

    def seq_pages(self, seq: int) -> np.ndarray:
        n = int(lib().hq_kv_pool_seq_pages(self._h, seq, None, 0))
        if n < 0:
            _bad(f"no sequence {seq}")
        out = np.empty(n, np.int32)
        lib().hq_kv_pool_seq_pages(self._h, seq, out.ctypes.data, n)
        return out

    def compact(self) -> list[tuple[int, int]]:
        """Renumbers the pages in use to 0 .. n-1; returns the page copies to make."""
        buf, n = np.empty((self.num_pages, 2), np.int32), ctypes.c_int(0)
        status = lib().hq_kv_pool_compact(self._h, buf.ctypes.data, self.num_pages, ctypes.byref(n))
        if status != _lib.HQ_OK:
            raise HQError(status, "compact")
        return [tuple(m) for m in buf[: n.value].tolist()]


class KVCache:
    """A paged cache of all layers: k and v [layers, num_pages, page_size, kv_heads, head_dim], and its pool."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16,
                 device="cuda"):
        self.pool = PagePool(num_pages, page_size)
        self.k = torch.zeros((layers, num_pages, page_size, kv_heads, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)

    def new_seq(self) -> int:
        return self.pool.new_seq()

    def fork(self, seq: int) -> int:
        return self.pool.fork(seq)

    def free(self, seq: int) -> None:
        self.pool.free(seq)

    def extend(self, seqs, counts, stream=None) -> None:
        """Room for counts[i] more keys of seqs[i]; pages that forks still share are copied, all layers in one call.
        Where the pages run out, the sequences before the failing one keep their room."""
        moves = []
        try:
            for s, n in zip(seqs, counts):
                moves += self.pool.extend(s, n)
        finally:
            self._copy(moves, stream)

    def compact(self, stream=None) -> int:
        """Moves the pages in use to the front; returns how many moved."""
        moves = self.pool.compact()
        self._copy(moves, stream)
        return len(moves)

    def _copy(self, moves, stream):
        if moves:
            kv_copy_pages([self.k, self.v], [m[0] for m in moves], [m[1] for m in moves], stream=stream)

    def tables(self, seqs) -> tuple[torch.Tensor, torch.Tensor, int]:
        """(page_table [n, pages] int32, kv_lens [n] int32, longest) of the sequences, on the cache's device."""
        lists = [self.pool.seq_pages(s) for s in seqs]
        lens = [self.pool.seq_len(s) for s in seqs]
        host = np.zeros((len(lists), max([len(p) for p in lists], default=0) + 1), np.int32)  # last column: lengths
        for row, p, n in zip(host, lists, lens):
            row[: len(p)] = p
            row[-1] = n
        dev = torch.from_numpy(host).to(self.k.device)
        return dev[:, :-1], dev[:, -1].contiguous(), max(lens, default=0)
