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
import operator
import struct
from array import array

import numpy as np
import torch

from . import _lib
from ._lib import HQ_BF16, HQ_F16, HQError, check, lib

__all__ = ["attn_prompt", "attn_paged", "kv_append", "kv_copy_pages", "PagePool", "KVCache"]

_DT = {torch.float16: HQ_F16, torch.bfloat16: HQ_BF16}

# The structures of include/hq.h as packed bytes: a call is shorter than building ctypes objects.
_ROWS = struct.Struct("@Pqq").pack                # hq_rows
_SHAPE = struct.Struct("@7if").pack               # hq_attn_shape
_VIEW = struct.Struct("@PqqqPqqqiiPqi4xP").pack   # hq_kv_view


def _bad(msg: str):
    raise HQError(_lib.HQ_ERR_INVALID_ARG, msg)


def _rows(t: torch.Tensor, name: str, dtype, dev: int, shape: tuple) -> bytes:
    """hq_rows of a [tokens, heads, head_dim] tensor."""
    if t.shape != shape:
        _bad(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype is not dtype or t.get_device() != dev:
        _bad(f"{name}: {t.dtype} on {t.device} beside {dtype} on device {dev}")
    st, sh, sd = t.stride()
    if sd != 1 and shape[2] > 1:
        _bad(f"{name}: head_dim must be contiguous")
    return _ROWS(t.data_ptr(), st, sh)


def _index(t: torch.Tensor | None, name: str, n: int, dev: int):
    """Device address of n contiguous int32 (None: null)."""
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.get_device() != dev or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        _bad(f"{name} must be {n} contiguous int32 on device {dev}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _view(k_pages, v_pages, page_table, kv_lens, dtype, dev: int, D: int) -> tuple:
    """(hq_kv_view, sequences, pages of a row of the table, page_size, kv_heads)."""
    shape = k_pages.shape
    if len(shape) != 4 or shape[3] != D:
        _bad(f"k_pages must be [num_pages, page_size, kv_heads, {D}], got {list(shape)}")
    if v_pages.shape != shape:
        _bad(f"key pages {list(shape)} and value pages {list(v_pages.shape)} differ")
    if k_pages.dtype is not dtype or v_pages.dtype is not dtype or k_pages.get_device() != dev or \
            v_pages.get_device() != dev:
        _bad(f"pages of {k_pages.dtype}, {v_pages.dtype} on {k_pages.device}, {v_pages.device} beside {dtype} on device {dev}")
    kp, kt, kh, kd = k_pages.stride()
    vp, vt, vh, vd = v_pages.stride()
    if (kd != 1 or vd != 1) and D > 1:
        _bad("pages: head_dim must be contiguous")
    table = page_table.shape
    if len(table) != 2 or page_table.dtype is not torch.int32 or page_table.get_device() != dev:
        _bad(f"page_table must be [sequences, pages] int32 on device {dev}")
    B, pages = table
    stride, inner = page_table.stride()
    if inner != 1 and pages > 1:
        _bad("page_table rows must be contiguous")
    return _VIEW(k_pages.data_ptr(), kp, kt, kh, v_pages.data_ptr(), vp, vt, vh, shape[0], shape[1], page_table.data_ptr(),
                 stride, pages, _index(kv_lens, "kv_lens", B, dev)), B, pages, shape[1], shape[2]


def _kind(q: torch.Tensor, what: str) -> tuple:
    """(dtype, its number, device) of [tokens, heads, head_dim] rows."""
    dtype, dev = q.dtype, q.get_device()
    dt = _DT.get(dtype)
    if dt is None:
        _bad(f"unsupported dtype {dtype}")
    if dev < 0:
        _bad(f"tensors must be on a CUDA device, got {q.device}")
    if q.dim() != 3:
        _bad(f"{what} must be [tokens, heads, head_dim], got {list(q.shape)}")
    return dtype, dt, dev


def _elsewhere(dev: int, stream):
    """None where device `dev` is current and the call goes on its current stream; else what makes it so (the call's
    allocations are then that stream's, too)."""
    if stream is not None:
        if stream.device.index != dev:
            _bad(f"a stream of {stream.device} for tensors on device {dev}")
        return torch.cuda.stream(stream)
    return None if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)


#: Handle of a device's current stream (torch.cuda.current_stream builds an object for it, ten times slower).
_raw_stream = torch._C._cuda_getCurrentRawStream


def _lse(lse, dev: int, shape: tuple):
    if lse is None:
        return None
    if lse.dtype is not torch.float32 or lse.shape != shape or not lse.is_contiguous() or lse.get_device() != dev:
        _bad(f"lse must be contiguous float32 {list(shape)} on device {dev}")
    return lse.data_ptr()


def _workspace(need: int, workspace, q: torch.Tensor, dev: int) -> tuple:
    """(tensor kept until the call is enqueued, address, bytes)."""
    if workspace is None:
        if not need:
            return None, None, 0
        workspace = q.new_empty(need // 2)
        return workspace, workspace.data_ptr(), need
    if workspace.get_device() != dev or not workspace.is_contiguous():
        _bad(f"workspace must be contiguous on device {dev}")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _output(out, q: torch.Tensor, dtype, dev: int, shape: tuple) -> tuple:
    """(tensor, hq_rows) of the output."""
    if out is not None:
        return out, _rows(out, "out", dtype, dev, shape)
    out = q.new_empty(shape)
    return out, _ROWS(out.data_ptr(), shape[1] * shape[2], shape[2])


def attn_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int, *,
                causal: bool = True, scale: float | None = None, out: torch.Tensor | None = None,
                lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention within packed sequences: q [T, Hq, D], k and v [T, Hkv, D]; sequence s is the rows
    cu_seqlens[s] .. cu_seqlens[s+1]-1, at most max_seqlen of them.  Rows behind the last sequence keep what `out`
    holds.  lse: optional [T, Hq] float32 output (ln of the softmax denominator)."""
    dtype, dt, dev = _kind(q, "q")
    ctx = _elsewhere(dev, stream)
    if ctx is not None:
        with ctx:
            return attn_prompt(q, k, v, cu_seqlens, max_seqlen, causal=causal, scale=scale, out=out, lse=lse,
                               workspace=workspace)
    if k.dim() != 3 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        _bad("k and v must be [tokens, kv_heads, head_dim], cu_seqlens [sequences + 1]")
    T, Hq, D = shape = q.shape
    Hk, B = k.shape[1], cu_seqlens.shape[0] - 1
    kv = (T, Hk, D)
    sh = _SHAPE(T, B, max_seqlen, Hq, Hk, D, dt, D ** -0.5 if scale is None else scale)
    out, ro = _output(out, q, dtype, dev, shape)
    L = lib()
    ws, ws_p, ws_n = _workspace(L.hq_attn_prompt_workspace_size(sh), workspace, q, dev)
    check(L.hq_attn_prompt(sh, _rows(q, "q", dtype, dev, shape), _rows(k, "k", dtype, dev, kv), _rows(v, "v", dtype, dev, kv),
                           _index(cu_seqlens, "cu_seqlens", B + 1, dev), int(causal), ro, _lse(lse, dev, (T, Hq)), ws_p, ws_n,
                           _raw_stream(dev)))
    return out


def attn_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
               kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, max_q_len: int = 1, *,
               max_kv_len: int | None = None, prefix_table: torch.Tensor | None = None, prefix_len: int = 0,
               scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention of a step's rows over a paged cache: q [T, Hq, D]; sequence s has the rows cu_q[s] .. cu_q[s+1]-1
    (cu_q None: row s alone), at most max_q_len, and kv_lens[s] keys, its rows' own last (kv_append writes them
    first).  Row i of n sees keys 0 .. kv_lens[s] - n + i, after the prefix_len keys of the pages prefix_table that
    every sequence shares.  max_kv_len: a bound of kv_lens by which the work is split (another one: the same results
    within rounding)."""
    dtype, dt, dev = _kind(q, "q")
    ctx = _elsewhere(dev, stream)
    if ctx is not None:
        with ctx:
            return attn_paged(q, k_pages, v_pages, page_table, kv_lens, cu_q, max_q_len, max_kv_len=max_kv_len,
                              prefix_table=prefix_table, prefix_len=prefix_len, scale=scale, out=out, lse=lse,
                              workspace=workspace)
    T, Hq, D = shape = q.shape
    view, B, pages, page_size, Hk = _view(k_pages, v_pages, page_table, kv_lens, dtype, dev, D)
    if max_kv_len is None:
        max_kv_len = pages * page_size
    pt = None
    if prefix_len:
        if prefix_table is None or prefix_table.dim() != 1 or prefix_table.shape[0] * page_size < prefix_len:
            _bad(f"prefix_table does not hold {prefix_len} keys")
        pt = _index(prefix_table, "prefix_table", prefix_table.shape[0], dev)
    sh = _SHAPE(T, B, max_q_len, Hq, Hk, D, dt, D ** -0.5 if scale is None else scale)
    out, ro = _output(out, q, dtype, dev, shape)
    L = lib()
    ws, ws_p, ws_n = _workspace(L.hq_attn_paged_workspace_size(sh, max_kv_len, prefix_len), workspace, q, dev)
    check(L.hq_attn_paged(sh, _rows(q, "q", dtype, dev, shape), view, _index(cu_q, "cu_q", B + 1, dev), max_kv_len, pt,
                          prefix_len, ro, _lse(lse, dev, (T, Hq)), ws_p, ws_n, _raw_stream(dev)))
    return out


def kv_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              page_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, *,
              stream=None) -> None:
    """Writes the rows of k and v [T, Hkv, D] into their pages: row i of the n rows of sequence s becomes its key
    kv_lens[s] - n + i."""
    dtype, dt, dev = _kind(k, "k")
    ctx = _elsewhere(dev, stream)
    if ctx is not None:
        with ctx:
            return kv_append(k, v, k_pages, v_pages, page_table, kv_lens, cu_q)
    T, Hk, D = shape = k.shape
    view, B, _, _, heads = _view(k_pages, v_pages, page_table, kv_lens, dtype, dev, D)
    if heads != Hk:
        _bad(f"{Hk} heads into pages of {heads}")
    check(lib().hq_kv_append(_SHAPE(T, B, T, Hk, Hk, D, dt, 1.0), _rows(k, "k", dtype, dev, shape),
                             _rows(v, "v", dtype, dev, shape), view, _index(cu_q, "cu_q", B + 1, dev), _raw_stream(dev)))


_I32 = np.dtype(np.int32)


def _int32(x, name: str) -> np.ndarray:
    """x as int32 one behind the other, without a number changed on the way."""
    if type(x) is list:  # a tenth of the time that numpy takes to look at one
        try:
            return np.asarray(array("i", x))
        except (TypeError, OverflowError):
            pass  # said below
    a = x if type(x) is np.ndarray else np.asarray(x)
    if a.dtype is _I32:
        return a if a.flags.c_contiguous else a.copy()
    if a.size and (a.dtype.kind not in "iub" or int(a.min()) < -2 ** 31 or int(a.max()) >= 2 ** 31):
        _bad(f"{name} must be integers that int32 holds, got {a.dtype} {a.reshape(-1)[:8].tolist()}")
    return a.astype(np.int32, order="C")


def _int(x, name: str) -> int:
    """x as an int of C's (ctypes takes the lower 32 bits of any)."""
    try:
        n = operator.index(x)
    except TypeError:
        n = None
    if n is None or not -2 ** 31 <= n < 2 ** 31:
        _bad(f"no {name} {x!r}")
    return n


def _moves(src, dst) -> bytes:
    """hq_page_move[n]."""
    n = len(src)
    if len(dst) != n:
        _bad(f"{n} source pages and {len(dst)} destinations")
    if isinstance(src, np.ndarray):
        both = np.empty((n, 2), _I32)
        both[:, 0] = src if src.dtype is _I32 else _int32(src, "source pages")
        both[:, 1] = dst if type(dst) is np.ndarray and dst.dtype is _I32 else _int32(dst, "destination pages")
    else:  # lists: half of what numpy takes, few moves or many
        both = array("i", bytes(8 * n))
        both[0::2] = array("i", src)
        both[1::2] = array("i", dst if not isinstance(dst, np.ndarray) else _int32(dst, "destination pages"))
    return both.tobytes()


def _page_bytes(shape, stride, size: int) -> int:
    """Bytes of a page whose dimensions lie, in some order, in one block."""
    run = 1
    for st, n in sorted(zip(stride, shape)):
        if n > 1:
            if st != run:
                _bad(f"a page must be one block of memory, got strides {tuple(stride)}")
            run *= n
    return run * size


def kv_copy_pages(pools, src, dst, *, stream=None) -> None:
    """Copies page src[i] over page dst[i] (host integers) in every pool: tensors [num_pages, ...] of four
    dimensions, or [layers, num_pages, ...] of five, all of one geometry, a page being one block of memory.  A page
    may be copied to several places; one that is written twice, or read and written, is refused."""
    both = _moves(src, dst)
    if not pools:
        return
    first = pools[0]
    dev = first.get_device()
    if dev < 0:
        _bad(f"pools must be on a CUDA device, got {first.device}")
    ctx = _elsewhere(dev, stream)
    if ctx is not None:
        with ctx:
            return kv_copy_pages(pools, src, dst)
    bases, geometry, last = [], None, None
    for t in pools:
        like = shape, stride, size = t.shape, t.stride(), t.element_size()
        if t.get_device() != dev or len(shape) not in (4, 5):
            _bad(f"pools must be on {first.device}, of 4 or 5 dimensions: got {list(shape)} on {t.device}")
        at = len(shape) - 4
        if like != last:
            g = (shape[at], stride[at] * size, _page_bytes(shape[at + 1:], stride[at + 1:], size))
            if geometry not in (None, g):
                _bad("pools of different geometry")
            geometry, last = g, like
        p = t.data_ptr()
        if at:
            step = stride[0] * size
            bases += [p + i * step for i in range(shape[0])]
        else:
            bases.append(p)
    check(lib().hq_kv_copy_pages(struct.pack(f"@{len(bases)}P", *bases), len(bases), geometry[1], geometry[2], geometry[0],
                                 both, len(src), _raw_stream(dev)))


class PagePool:
    """Pages of a cache by sequence: reference counts and page lists on the host (hq_kv_pool_*)."""

    def __init__(self, num_pages: int, page_size: int):
        self._h = None
        num_pages, page_size = _int(num_pages, "number of pages"), _int(page_size, "page size")
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
        s = int(lib().hq_kv_pool_fork(self._h, _int(seq, "sequence")))
        if s < 0:
            _bad(f"no sequence {seq}")
        return s

    def extend(self, seqs, counts) -> list[tuple[int, int]]:
        """Room for counts[i] more keys of seqs[i] (integers, or lists of them), for all or for none; returns the page
        copies, (source, destination), to make first."""
        seqs, counts = np.atleast_1d(_int32(seqs, "sequences")), np.atleast_1d(_int32(counts, "counts"))
        if seqs.ndim != 1 or seqs.shape != counts.shape:
            _bad(f"{seqs.size} sequences and {counts.size} counts")
        moves, n = np.empty((max(1, seqs.size), 2), np.int32), ctypes.c_int(0)
        status = lib().hq_kv_pool_extend(self._h, seqs.ctypes.data, counts.ctypes.data, seqs.size, moves.ctypes.data,
                                         ctypes.byref(n))
        if status != _lib.HQ_OK:
            raise HQError(status, f"sequences {seqs.tolist()} by {counts.tolist()} keys, {self.free_pages} pages free")
        return [tuple(m) for m in moves[: n.value].tolist()]

    def free(self, seq: int) -> None:
        status = lib().hq_kv_pool_free(self._h, _int(seq, "sequence"))
        if status != _lib.HQ_OK:
            raise HQError(status, f"no sequence {seq}")

    def seq_len(self, seq: int) -> int:
        n = int(lib().hq_kv_pool_seq_len(self._h, _int(seq, "sequence")))
        if n < 0:
            _bad(f"no sequence {seq}")
        return n

    def seq_pages(self, seq: int) -> np.ndarray:
        seq = _int(seq, "sequence")
        n = int(lib().hq_kv_pool_seq_pages(self._h, seq, None, 0))
        if n < 0:
            _bad(f"no sequence {seq}")
        out = np.empty(n, np.int32)
        lib().hq_kv_pool_seq_pages(self._h, seq, out.ctypes.data, n)
        return out

    def tables(self, seqs) -> tuple[np.ndarray, np.ndarray]:
        """(page table [n, pages], lengths [n]) of the sequences, int32 on the host."""
        seqs = _int32(seqs, "sequences").reshape(-1)
        L, lens = lib(), np.empty(seqs.size, np.int32)
        pages = int(L.hq_kv_pool_tables(self._h, seqs.ctypes.data, seqs.size, None, 0, lens.ctypes.data))
        if pages < 0:
            _bad(f"no such sequence among {seqs.tolist()}")
        table = np.empty((seqs.size, pages), np.int32)
        L.hq_kv_pool_tables(self._h, seqs.ctypes.data, seqs.size, table.ctypes.data, pages, None)
        return table, lens

    def compact(self) -> list[tuple[int, int]]:
        """Renumbers the pages in use to 0 .. n-1; returns the page copies to make."""
        buf, n = np.empty((self.num_pages, 2), np.int32), ctypes.c_int(0)
        status = lib().hq_kv_pool_compact(self._h, buf.ctypes.data, self.num_pages, ctypes.byref(n))
        if status != _lib.HQ_OK:
            raise HQError(status, "compact")
        return [tuple(m) for m in buf[: n.value].tolist()]


class KVCache:
    """A paged cache of all layers: k and v [layers, num_pages, page_size, kv_heads, head_dim], and its pool.  The page
    copies of an extend or compact that raised are made by the next one, before its own."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16,
                 device="cuda"):
        self.pool = PagePool(num_pages, page_size)
        self.k = torch.zeros((layers, num_pages, page_size, kv_heads, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self._owed = []  # lists of copies that the pool counts on, in their order

    def new_seq(self) -> int:
        return self.pool.new_seq()

    def fork(self, seq: int) -> int:
        return self.pool.fork(seq)

    def free(self, seq: int) -> None:
        self.pool.free(seq)

    def extend(self, seqs, counts, stream=None) -> None:
        """Room for counts[i] more keys of seqs[i], for all or for none; pages that forks still share are copied, all
        layers in one call."""
        self._move(self.pool.extend(seqs, counts), stream)

    def compact(self, stream=None) -> int:
        """Moves the pages in use to the front; returns how many moved."""
        moves = self.pool.compact()
        self._move(moves, stream)
        return len(moves)

    def _move(self, moves, stream):
        self._owed.append(moves)
        while self._owed:
            self._copy(self._owed[0], stream)
            del self._owed[0]

    def _copy(self, moves, stream):
        if moves:
            kv_copy_pages([self.k, self.v], [m[0] for m in moves], [m[1] for m in moves], stream=stream)

    def tables(self, seqs) -> tuple[torch.Tensor, torch.Tensor, int]:
        """(page_table [n, pages] int32, kv_lens [n] int32, longest) of the sequences, on the cache's device."""
        table, lens = self.pool.tables(seqs)
        dev = torch.from_numpy(np.concatenate([table.reshape(-1), lens])).to(self.k.device)  # one copy for both
        return dev[: table.size].view(table.shape), dev[table.size:], int(lens.max(initial=0))
