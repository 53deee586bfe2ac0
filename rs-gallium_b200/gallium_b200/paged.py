"""The paged KV cache's operators over the C ABI (gb_paged_*), on torch CUDA
tensors, and a host-side page allocator.

A pool is a tensor of [n_pages, page_size, n_kv_heads, head_dim] (any strides
whose last dimension is contiguous, so a [page][head][slot][dim] pool is a
transposed view), bf16 or f16; ``PagedBatch`` describes the ragged batch that
a step works on and serves all layers of it.  Every call runs on torch's
current stream of the tensors' device and synchronises nothing:
``PagedBatch.check`` reads what the kernels flagged.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence

from . import _lib
from ._lib import AttnArgs, GalliumError, PagedBatchDesc, RopeArgs, load_library

_DTYPES = None


def _dtype(t) -> int:
    global _DTYPES
    if _DTYPES is None:
        import torch

        _DTYPES = {torch.float32: _lib.GB_DTYPE_F32, torch.bfloat16: _lib.GB_DTYPE_BF16,
                   torch.float16: _lib.GB_DTYPE_F16}
    d = _DTYPES.get(t)
    if d is None:
        raise GalliumError(_lib.GB_ERR_UNSUPPORTED, f"dtype {t}: float32, bfloat16 or float16")
    return d


def _bad(message: str):
    raise GalliumError(_lib.GB_ERR_INVALID_ARG, message)


def _check(rc: int) -> None:
    if rc:
        _lib.check(rc)


def _on(device, name, t):
    if t.device != device:
        _bad(f"{name} is on {t.device}, the batch on {device}")


class _Call:
    """The device's current stream, with that device current during the call."""

    def __init__(self, device):
        import torch

        self._guard = torch.cuda.device(device) if torch.cuda.current_device() != device.index else None
        self.stream = torch.cuda.current_stream(device).cuda_stream

    def __enter__(self):
        if self._guard is not None:
            self._guard.__enter__()
        return self.stream

    def __exit__(self, *exc):
        if self._guard is not None:
            self._guard.__exit__(*exc)


class PagedBatch:
    """A ragged batch of new tokens over the pages of their sequences.

    q_start (n_seqs + 1,) int32, kv_len (n_seqs,) int32 with the new tokens,
    page_table (n_seqs, entries) int32, all on one CUDA device, read by the
    kernels when they run: a captured graph sees their contents at replay, so
    long as they keep within total_q (rows of q), max_q_len and max_kv_len.
    The tensors are used as they are (no copies) and must be contiguous; rows
    of page_table may be strided.
    """

    def __init__(self, q_start, kv_len, page_table, *, page_size: int, total_q: int, max_q_len: int,
                 max_kv_len: int):
        import torch

        for name, t, nd in (("q_start", q_start, 1), ("kv_len", kv_len, 1), ("page_table", page_table, 2)):
            if t.dtype != torch.int32 or t.dim() != nd or not t.is_cuda:
                _bad(f"{name} must be an int32 CUDA tensor of {nd} dimension(s)")
            _on(q_start.device, name, t)
        n = kv_len.shape[0]
        if q_start.shape[0] != n + 1 or page_table.shape[0] != n:
            _bad(f"q_start needs {n + 1} entries and page_table {n} rows")
        if not q_start.is_contiguous() or not kv_len.is_contiguous() or (
                page_table.shape[1] > 1 and page_table.stride(1) != 1):
            _bad("q_start, kv_len and the rows of page_table must be contiguous")
        if n > 1 and page_table.stride(0) < page_table.shape[1]:
            _bad("the rows of page_table must not overlap")
        self.q_start, self.kv_len, self.page_table = q_start, kv_len, page_table
        self.device = q_start.device
        self.error = torch.zeros(1, dtype=torch.int32, device=self.device)
        d = PagedBatchDesc()
        d.struct_size = ctypes.sizeof(PagedBatchDesc)
        d.page_size = page_size
        d.n_seqs, d.total_q = n, total_q
        d.max_q_len, d.max_kv_len = max_q_len, max_kv_len
        d.q_start_dev, d.kv_len_dev = q_start.data_ptr(), kv_len.data_ptr()
        d.page_table_dev = page_table.data_ptr()
        d.table_stride = page_table.stride(0) if n > 1 else page_table.shape[1]
        if n > 1 and d.table_stride != page_table.shape[1]:
            # kernels bound a position by table_stride entries: keep them inside the tensor
            d.max_kv_len = min(max_kv_len, page_table.shape[1] * page_size)
        d.error_dev = self.error.data_ptr()
        self._desc = d
        self._ref = ctypes.byref(d)
        self._workspace = {}
        self._pool = None

    @property
    def total_q(self) -> int:
        return self._desc.total_q

    def check(self) -> None:
        """Raises GalliumError when a kernel of this batch flagged its device
        arrays since the last check (gb_paged_error).  Synchronises."""
        bits = int(self.error.item())
        if not bits:
            return
        self.error.zero_()
        what = [text for bit, text in ((1, "a needed page number is outside the pool"),
                                       (2, "q_start or kv_len is outside its bounds"),
                                       (4, "a position is outside the rotation tables"),
                                       (8, "a pipeline wait ran out")) if bits & bit]
        raise GalliumError(_lib.GB_ERR_TIMEOUT if bits & 8 else _lib.GB_ERR_INVALID_ARG, "; ".join(what))

    def _set_pool(self, k_pool, v_pool) -> None:
        """Puts the pools' shape, strides and type into the descriptor."""
        key = (k_pool.shape, k_pool.stride(), k_pool.dtype)
        if v_pool.shape != key[0] or v_pool.stride() != key[1] or v_pool.dtype != key[2]:
            _bad("the K and V pools differ in shape, strides or dtype")
        _on(self.device, "k_pool", k_pool)
        _on(self.device, "v_pool", v_pool)
        if key == self._pool:
            return
        if k_pool.dim() != 4 or k_pool.shape[1] != self._desc.page_size or (
                k_pool.shape[3] > 1 and k_pool.stride(3) != 1):
            _bad(f"a pool is [n_pages, {self._desc.page_size}, n_kv_heads, head_dim] with a contiguous last "
                 f"dimension, got {tuple(k_pool.shape)} with strides {k_pool.stride()}")
        d = self._desc
        d.dtype = _dtype(k_pool.dtype)
        d.n_pages, _, d.n_kv_heads, d.head_dim = k_pool.shape
        d.page_stride, d.slot_stride, d.head_stride, _ = k_pool.stride()
        self._pool = key

    def _workspace_bytes(self, n_heads: int) -> int:
        key = (n_heads, self._desc.n_kv_heads, self._desc.head_dim)
        got = self._workspace.get(key)
        if got is None:
            n = ctypes.c_int64()
            _check(load_library().gb_paged_attention_workspace(self._ref, n_heads, ctypes.byref(n)))
            got = self._workspace[key] = n.value
        return got


def _rows(name, x, batch, heads, dim):
    if x.dim() != 3 or x.shape[0] != batch.total_q or (heads is not None and x.shape[1] != heads) or (
            x.shape[2] != dim) or (dim > 1 and x.stride(2) != 1):
        _bad(f"{name} must be [{batch.total_q}, {heads or 'heads'}, {dim}] with a contiguous last dimension, "
             f"got {tuple(x.shape)} with strides {x.stride()}")
    _on(batch.device, name, x)


def rope_append(batch: PagedBatch, q, k, v, k_pool, v_pool, cos=None, sin=None, *, q_norm=None, k_norm=None,
                eps: float = 1e-6, q_out=None):
    """RMS norm of each query and key head (where q_norm / k_norm (head_dim,)
    f32 are given), rotation by the rows' positions (cos, sin (positions,
    rot_dim / 2) f32; None: none), k and v stored into their pages.  q, k, v
    [total_q, heads, head_dim] f32, bf16 or f16, any row and head strides.
    Returns the queries in the pools' dtype (q_out, when given; q itself is
    allowed when the dtypes agree).  Rows of no sequence keep q_out's values."""
    import torch

    batch._set_pool(k_pool, v_pool)
    d = batch._desc
    _rows("q", q, batch, None, d.head_dim)
    _rows("k", k, batch, d.n_kv_heads, d.head_dim)
    _rows("v", v, batch, d.n_kv_heads, d.head_dim)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        _bad("q, k and v must have one dtype")
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=k_pool.dtype, device=batch.device)
    else:
        _rows("q_out", q_out, batch, q.shape[1], d.head_dim)
        if q_out.dtype != k_pool.dtype:
            _bad(f"q_out must be {k_pool.dtype}")
    a = RopeArgs()
    a.struct_size = ctypes.sizeof(RopeArgs)
    if (cos is None) != (sin is None):
        _bad("cos and sin come together")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None:
            if w.dtype != torch.float32 or w.shape != (d.head_dim,) or not w.is_contiguous():
                _bad(f"{name} must be a contiguous float32 ({d.head_dim},)")
            _on(batch.device, name, w)
    if cos is not None:
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or (
                cos.shape != sin.shape) or not cos.is_contiguous() or not sin.is_contiguous():
            _bad("cos and sin must be contiguous float32 (positions, rot_dim / 2)")
        _on(batch.device, "cos", cos)
        _on(batch.device, "sin", sin)
        a.rot_dim, a.table_rows = 2 * cos.shape[1], cos.shape[0]
        a.cos_dev, a.sin_dev = cos.data_ptr(), sin.data_ptr()
    a.in_dtype, a.n_heads, a.eps = _dtype(q.dtype), q.shape[1], eps
    a.q_dev, a.k_dev, a.v_dev, a.q_out_dev = q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr()
    a.q_row_stride, a.q_head_stride, _ = q.stride()
    a.k_row_stride, a.k_head_stride, _ = k.stride()
    a.v_row_stride, a.v_head_stride, _ = v.stride()
    a.out_row_stride, a.out_head_stride, _ = q_out.stride()
    if q_norm is not None:
        a.q_norm_dev = q_norm.data_ptr()
    if k_norm is not None:
        a.k_norm_dev = k_norm.data_ptr()
    a.k_pool_dev, a.v_pool_dev = k_pool.data_ptr(), v_pool.data_ptr()
    with _Call(batch.device) as stream:
        _check(load_library().gb_paged_rope_append(batch._ref, ctypes.byref(a), stream))
    return q_out


def attention(batch: PagedBatch, q, k_pool, v_pool, *, sinks=None, window: int = 0,
              scale: Optional[float] = None, out=None):
    """Causal attention of q [total_q, n_heads, head_dim] (the pools' dtype)
    over the sequences' pages; window > 0: the last `window` positions only;
    sinks (n_heads,) f32: a sink logit per head; scale defaults to
    head_dim^-1/2.  Returns out (q's shape; the pools' dtype, or float32 when
    such an `out` is given).  Rows of no sequence keep out's values."""
    import torch

    batch._set_pool(k_pool, v_pool)
    d = batch._desc
    _rows("q", q, batch, None, d.head_dim)
    if q.dtype != k_pool.dtype:
        _bad(f"q must be {k_pool.dtype}, as the pools")
    heads = q.shape[1]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=batch.device)
    else:
        _rows("out", out, batch, heads, d.head_dim)
    if sinks is not None:
        if sinks.dtype != torch.float32 or sinks.shape != (heads,) or not sinks.is_contiguous():
            _bad(f"sinks must be a contiguous float32 ({heads},)")
        _on(batch.device, "sinks", sinks)
    a = AttnArgs()
    a.struct_size = ctypes.sizeof(AttnArgs)
    a.n_heads, a.window, a.out_dtype = heads, window, _dtype(out.dtype)
    a.scale = d.head_dim ** -0.5 if scale is None else scale
    a.q_dev, a.out_dev = q.data_ptr(), out.data_ptr()
    a.q_row_stride, a.q_head_stride, _ = q.stride()
    a.out_row_stride, a.out_head_stride, _ = out.stride()
    a.k_pool_dev, a.v_pool_dev = k_pool.data_ptr(), v_pool.data_ptr()
    if sinks is not None:
        a.sinks_dev = sinks.data_ptr()
    a.workspace_bytes = batch._workspace_bytes(heads)
    with _Call(batch.device) as stream:
        # torch's allocator orders the workspace's next use after this stream's work
        ws = torch.empty(a.workspace_bytes, dtype=torch.uint8, device=batch.device)
        a.workspace_dev = ws.data_ptr()
        _check(load_library().gb_paged_attention(batch._ref, ctypes.byref(a), stream))
    return out


def copy_pages(pools, src: Sequence[int], dst: Sequence[int]) -> None:
    """Copies page src[i] to page dst[i] in every pool: `pools` is one tensor
    [n_pools, n_pages, ...] or a sequence of tensors [n_pages, ...] of one
    shape, dtype and strides, whose pages are dense (a page's elements fill one
    block of memory).  src and dst are host integers; a page may be copied to
    several others, none may be written twice or both read and written."""
    import torch

    if len(src) != len(dst):
        _bad("src and dst differ in length")
    if torch.is_tensor(pools):
        one, n_pools = pools[0] if pools.shape[0] else None, pools.shape[0]
    else:
        n_pools = len(pools)
        one = pools[0] if n_pools else None
        for p in pools:
            if p.shape != one.shape or p.stride() != one.stride() or p.dtype != one.dtype or (
                    p.device != one.device):
                _bad("the pools differ in shape, strides, dtype or device")
    if one is None:
        return
    if not one.is_cuda or one.dim() < 2:
        _bad("a pool is a CUDA tensor of [n_pages, ...]")
    elems = one[0].numel()
    dense = 1
    for size, stride in sorted(((z, s) for z, s in zip(one.shape[1:], one.stride()[1:]) if z > 1),
                               key=lambda v: v[1]):
        if stride != dense:
            _bad(f"a pool's pages must be dense, got shape {tuple(one.shape)} with strides {one.stride()}")
        dense *= size
    size = one.element_size()
    page_stride = one.stride(0) * size if one.shape[0] > 1 else elems * size
    if torch.is_tensor(pools):
        step, base = pools.stride(0) * size, pools.data_ptr()
        ptrs = (ctypes.c_void_p * n_pools)(*[base + i * step for i in range(n_pools)])
    else:
        ptrs = (ctypes.c_void_p * n_pools)(*[p.data_ptr() for p in pools])
    n = len(src)
    s, t = (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst)
    with _Call(one.device) as stream:
        _check(load_library().gb_paged_copy(ptrs, n_pools, one.shape[0], elems * size, page_stride, s, t, n,
                                            stream))


class PagePool:
    """Host-side allocator of a paged cache's pages: which pages each sequence
    holds, shared pages by reference count.  It owns no device memory: the
    page moves that an operation needs are returned as (src, dst) lists for
    ``copy_pages``, which goes over every layer's pools before the next use of
    the pages it names."""

    def __init__(self, n_pages: int, page_size: int):
        if n_pages < 1 or page_size < 1:
            _bad("n_pages and page_size must be >= 1")
        self.page_size = page_size
        self._refs = [0] * n_pages
        self._free = list(range(n_pages - 1, -1, -1))  # the lowest page is handed out first
        self._seqs = {}
        self._next = 0

    @property
    def n_free(self) -> int:
        return len(self._free)

    def pages(self, seq: int) -> List[int]:
        return list(self._get(seq)[0])

    def length(self, seq: int) -> int:
        return self._get(seq)[1]

    def _get(self, seq):
        if seq not in self._seqs:
            _bad(f"no sequence {seq}")
        return self._seqs[seq]

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if not self._refs[page]:
            self._free.append(page)

    def add(self) -> int:
        """A new, empty sequence."""
        self._next += 1
        self._seqs[self._next] = [[], 0]
        return self._next

    def extend(self, seq: int, n_tokens: int):
        """Room for n_tokens more; returns the (src, dst) copies that must run
        before they are written: a last page that a fork shares is replaced by
        a copy.  GB_ERR_NO_MEMORY, nothing changed, when the pages are out."""
        if n_tokens < 0:
            _bad("n_tokens < 0")
        entry = self._get(seq)
        pages, length = entry
        partial = length % self.page_size
        split = n_tokens > 0 and partial and self._refs[pages[-1]] > 1
        need = -(-(length + n_tokens) // self.page_size) - len(pages) + (1 if split else 0)
        if need > len(self._free):
            raise GalliumError(_lib.GB_ERR_NO_MEMORY, f"{need} pages needed, {len(self._free)} free")
        src, dst = [], []
        if split:
            old = pages[-1]
            pages[-1] = self._take()
            self._drop(old)
            src.append(old)
            dst.append(pages[-1])
            need -= 1
        pages.extend(self._take() for _ in range(need))
        entry[1] = length + n_tokens
        return src, dst

    def fork(self, seq: int) -> int:
        """A sequence with the same tokens; pages are shared until extended."""
        pages, length = self._get(seq)
        for p in pages:
            self._refs[p] += 1
        new = self.add()
        self._seqs[new] = [list(pages), length]
        return new

    def truncate(self, seq: int, length: int) -> None:
        """Forgets the tokens at and past `length` and frees their pages."""
        entry = self._get(seq)
        if not 0 <= length <= entry[1]:
            _bad(f"length {length} outside [0, {entry[1]}]")
        keep = -(-length // self.page_size)
        for p in entry[0][keep:]:
            self._drop(p)
        del entry[0][keep:]
        entry[1] = length

    def free(self, seq: int) -> None:
        for p in self._get(seq)[0]:
            self._drop(p)
        del self._seqs[seq]

    def compact(self):
        """Moves the held pages to the lowest page numbers; returns the (src,
        dst) copies.  The pages from n_pages - n_free on are free after it."""
        held = len(self._refs) - len(self._free)
        holes = sorted(p for p in self._free if p < held)
        high = [p for p in range(held, len(self._refs)) if self._refs[p]]
        moved = dict(zip(high, holes))
        for a, b in moved.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        for entry in self._seqs.values():
            entry[0][:] = [moved.get(p, p) for p in entry[0]]
        self._free = list(range(len(self._refs) - 1, held - 1, -1))
        return list(moved), list(moved.values())

    def table(self, seqs: Sequence[int], width: Optional[int] = None):
        """The sequences' page numbers as an int32 array (len(seqs), width),
        unused entries -1."""
        import numpy as np

        rows = [self._get(s)[0] for s in seqs]
        need = max([len(r) for r in rows] + [1])
        width = need if width is None else width
        if width < need:
            _bad(f"width {width}: {need} pages needed")
        t = np.full((len(rows), width), -1, np.int32)
        for i, r in enumerate(rows):
            t[i, :len(r)] = r
        return t
