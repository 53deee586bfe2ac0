"""The paged KV cache's operators over the C ABI (gb_paged_*), on torch CUDA
tensors, and a host-side page allocator.

A pool is a tensor of [n_pages, page_size, n_kv_heads, head_dim] (any strides
whose last dimension is contiguous, so a [page][head][slot][dim] pool is a
transposed view), bf16 or f16; ``PagedBatch`` describes the ragged batch that
a step works on and serves all layers of it.  Every call runs on torch's
current stream of the tensors' device and synchronises nothing:
``PagedBatch.check`` reads what the kernels flagged.  There is no backward
form: results carry no graph, whether or not an input requires a gradient.
"""
from __future__ import annotations

import ctypes
from array import array
from typing import List, Optional, Sequence

from . import _lib
from ._lib import AttnArgs, GalliumError, PagedBatchDesc, RopeArgs, load_library

_ROPE_SIZE, _ATTN_SIZE = ctypes.sizeof(RopeArgs), ctypes.sizeof(AttnArgs)

torch = None  # imported by the first call: the package loads without it
_DTYPES = {}
_lib_handle = None


def _start():
    global torch, _lib_handle
    if _lib_handle is None:
        import torch as t

        torch = t
        _DTYPES.update({t.float32: _lib.GB_DTYPE_F32, t.bfloat16: _lib.GB_DTYPE_BF16,
                        t.float16: _lib.GB_DTYPE_F16})
        _lib_handle = load_library()
    return _lib_handle


def _dtype(t) -> int:
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
        _bad(f"{name} is on {t.device}, not on {device}")


def _call(fn, device, *args) -> None:
    """fn(*args, stream) on the device's current stream, that device current during the call."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)  # torch.cuda.current_stream without the Stream object
    if torch.cuda.current_device() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


class PagedBatch:
    """A ragged batch of new tokens over the pages of their sequences.

    q_start (n_seqs + 1,) int32, kv_len (n_seqs,) int32 with the new tokens,
    page_table (n_seqs, entries) int32, all on one CUDA device, read by the
    kernels when they run: a captured graph sees their contents at replay, so
    long as they keep within total_q (rows of q), max_q_len and max_kv_len.
    The tensors are used as they are (no copies) and must be contiguous; rows
    of page_table may be strided.

    The error word is zeroed here, on the current stream, and read and zeroed by
    check() on the stream current then: calls on another stream are ordered after
    the one and before the other by the caller, like the tensors above, or a flag
    may be lost.  A batch holds the descriptor of the call being made, so two
    threads take one each.
    """

    def __init__(self, q_start, kv_len, page_table, *, page_size: int, total_q: int, max_q_len: int,
                 max_kv_len: int):
        _start()
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
        self.total_q = total_q
        self._desc = d
        self._ref = ctypes.byref(d)
        self._workspace = {}
        self._pool = None

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
        shape, strides, dtype = k_pool.shape, k_pool.stride(), k_pool.dtype
        if v_pool.shape != shape or v_pool.stride() != strides or v_pool.dtype != dtype:
            _bad("the K and V pools differ in shape, strides or dtype")
        _on(self.device, "k_pool", k_pool)
        _on(self.device, "v_pool", v_pool)
        was = self._pool
        if was is not None and was[0] == shape and was[1] == strides and was[2] == dtype:
            return
        d = self._desc
        if len(shape) != 4 or shape[1] != d.page_size or (shape[3] > 1 and strides[3] != 1):
            _bad(f"a pool is [n_pages, {d.page_size}, n_kv_heads, head_dim] with a contiguous last "
                 f"dimension, got {tuple(shape)} with strides {strides}")
        d.dtype = _dtype(dtype)
        d.n_pages, _, d.n_kv_heads, d.head_dim = shape
        d.page_stride, d.slot_stride, d.head_stride, _ = strides
        self._pool = (shape, strides, dtype)

    def _workspace_bytes(self, n_heads: int) -> int:
        key = (n_heads, self._desc.n_kv_heads, self._desc.head_dim)
        got = self._workspace.get(key)
        if got is None:
            n = ctypes.c_int64()
            _check(_lib_handle.gb_paged_attention_workspace(self._ref, n_heads, ctypes.byref(n)))
            got = self._workspace[key] = n.value
        return got


def _rows(name, x, batch, heads, dim):
    """The row and head strides of x [total_q, heads, dim]."""
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != batch.total_q or shape[2] != dim or strides[2] != 1 or (
            heads is not None and shape[1] != heads):
        _bad(f"{name} must be [{batch.total_q}, {'heads' if heads is None else heads}, {dim}] with a "
             f"contiguous last dimension, got {tuple(shape)} with strides {strides}")
    if x.device != batch.device:
        _on(batch.device, name, x)
    return strides


def _vector(name, x, n, device, dtype=None):
    """The address of x, a contiguous vector of n values (float32 by default)."""
    dtype = dtype or torch.float32
    if x.dtype != dtype or x.dim() != 1 or x.shape[0] != n or not x.is_contiguous():
        _bad(f"{name} must be a contiguous {dtype} ({n},)")
    if x.device != device:
        _on(device, name, x)
    return x.data_ptr()


def rope_append(batch: PagedBatch, q, k, v, k_pool, v_pool, cos=None, sin=None, *, q_norm=None, k_norm=None,
                eps: float = 1e-6, q_out=None):
    """RMS norm of each query and key head (where q_norm / k_norm (head_dim,)
    f32 are given), rotation by the rows' positions (cos, sin (positions,
    rot_dim / 2) f32; None: none), k and v stored into their pages.  q, k, v
    [total_q, heads, head_dim] f32, bf16 or f16, any row and head strides.
    Returns the queries in the pools' dtype (q_out, when given; q itself is
    allowed when the dtypes agree).  Rows of no sequence keep q_out's values."""
    batch._set_pool(k_pool, v_pool)
    d = batch._desc
    dim, device = d.head_dim, batch.device
    a = RopeArgs()
    a.q_row_stride, a.q_head_stride, _ = _rows("q", q, batch, None, dim)
    a.k_row_stride, a.k_head_stride, _ = _rows("k", k, batch, d.n_kv_heads, dim)
    a.v_row_stride, a.v_head_stride, _ = _rows("v", v, batch, d.n_kv_heads, dim)
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype:
        _bad("q, k and v must have one dtype")
    heads = q.shape[1]
    if q_out is None:
        q_out = torch.empty_like(q, dtype=k_pool.dtype)
        a.out_row_stride, a.out_head_stride, _ = q_out.stride()
    else:
        a.out_row_stride, a.out_head_stride, _ = _rows("q_out", q_out, batch, heads, dim)
        if q_out.dtype != k_pool.dtype:
            _bad(f"q_out must be {k_pool.dtype}")
    a.struct_size = _ROPE_SIZE
    if cos is not None and sin is not None:
        shape = cos.shape
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(shape) != 2 or (
                sin.shape != shape) or not cos.is_contiguous() or not sin.is_contiguous():
            _bad("cos and sin must be contiguous float32 (positions, rot_dim / 2)")
        _on(device, "cos", cos)
        _on(device, "sin", sin)
        a.rot_dim, a.table_rows = 2 * shape[1], shape[0]
        a.cos_dev, a.sin_dev = cos.data_ptr(), sin.data_ptr()
    elif cos is not None or sin is not None:
        _bad("cos and sin come together")
    if q_norm is not None:
        a.q_norm_dev = _vector("q_norm", q_norm, dim, device)
    if k_norm is not None:
        a.k_norm_dev = _vector("k_norm", k_norm, dim, device)
    a.in_dtype, a.n_heads, a.eps = _dtype(dtype), heads, eps
    a.q_dev, a.k_dev, a.v_dev, a.q_out_dev = q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr()
    a.k_pool_dev, a.v_pool_dev = k_pool.data_ptr(), v_pool.data_ptr()
    _call(_lib_handle.gb_paged_rope_append, device, batch._ref, ctypes.byref(a))
    return q_out


def attention(batch: PagedBatch, q, k_pool, v_pool, *, sinks=None, window: int = 0,
              scale: Optional[float] = None, out=None):
    """Causal attention of q [total_q, n_heads, head_dim] (the pools' dtype)
    over the sequences' pages; window > 0: the last `window` positions only;
    sinks (n_heads,) f32: a sink logit per head; scale defaults to
    head_dim^-1/2.  Returns out (q's shape; the pools' dtype, or float32 when
    such an `out` is given).  Rows of no sequence keep out's values."""
    batch._set_pool(k_pool, v_pool)
    d = batch._desc
    dim, device = d.head_dim, batch.device
    a = AttnArgs()
    a.q_row_stride, a.q_head_stride, _ = _rows("q", q, batch, None, dim)
    if q.dtype != k_pool.dtype:
        _bad(f"q must be {k_pool.dtype}, as the pools")
    heads = q.shape[1]
    if out is None:
        out = torch.empty_like(q)
        a.out_row_stride, a.out_head_stride, _ = out.stride()
        a.out_dtype = d.dtype
    else:
        a.out_row_stride, a.out_head_stride, _ = _rows("out", out, batch, heads, dim)
        a.out_dtype = _dtype(out.dtype)
    if sinks is not None:
        a.sinks_dev = _vector("sinks", sinks, heads, device)
    a.struct_size = _ATTN_SIZE
    a.n_heads, a.window = heads, window
    a.scale = dim ** -0.5 if scale is None else scale
    a.q_dev, a.out_dev = q.data_ptr(), out.data_ptr()
    a.k_pool_dev, a.v_pool_dev = k_pool.data_ptr(), v_pool.data_ptr()
    a.workspace_bytes = size = batch._workspace_bytes(heads)
    # torch's allocator orders the workspace's next use after this stream's work
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    a.workspace_dev = workspace.data_ptr()
    _call(_lib_handle.gb_paged_attention, device, batch._ref, ctypes.byref(a))
    return out


def copy_pages(pools, src: Sequence[int], dst: Sequence[int]) -> None:
    """Copies page src[i] to page dst[i] in every pool: `pools` is one tensor
    [n_pools, n_pages, ...] or a sequence of tensors [n_pages, ...] of one
    shape, dtype and strides, whose pages are dense (a page's elements fill one
    block of memory).  src and dst are host integers; a page may be copied to
    several others, none may be written twice or both read and written."""
    lib = _start()
    n = len(src)
    if n != len(dst):
        _bad("src and dst differ in length")
    if torch.is_tensor(pools):
        one, n_pools = pools, pools.shape[0]
        shape, strides = pools.shape[1:], pools.stride()[1:]
    else:
        n_pools = len(pools)
        if not n_pools:
            return
        one = pools[0]
        shape, strides, dtype, device = one.shape, one.stride(), one.dtype, one.device
        for p in pools:
            if p.shape != shape or p.stride() != strides or p.dtype != dtype or p.device != device:
                _bad("the pools differ in shape, strides, dtype or device")
    if not one.is_cuda or len(shape) < 2:
        _bad("a pool is a CUDA tensor of [n_pages, ...]")
    dense = 1
    for stride, extent in sorted(zip(strides[1:], shape[1:])):
        if extent > 1 and stride != dense:
            _bad(f"a pool's pages must be dense, got shape {tuple(shape)} with strides {strides}")
        dense *= extent
    size = one.element_size()
    page_stride = strides[0] * size if shape[0] > 1 else dense * size
    if one is pools:
        step, base = pools.stride(0) * size, pools.data_ptr()
        ptrs = array("Q", [base + i * step for i in range(n_pools)])
    else:
        ptrs = array("Q", [p.data_ptr() for p in pools])
    try:
        s, t = array("i", src), array("i", dst)
    except (OverflowError, TypeError) as e:
        _bad(f"src and dst must be 32-bit integers: {e}")
    _call(lib.gb_paged_copy, one.device, ptrs.buffer_info()[0], n_pools, shape[0], dense * size, page_stride,
          s.buffer_info()[0], t.buffer_info()[0], n)


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
