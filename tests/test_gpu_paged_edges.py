"""The attention of paged caches where its inputs are at their worst: device arrays
that contradict themselves, values that are not finite, rows beside rows.  Batches
and tolerances are those of test_gpu_paged.py."""
import ctypes

import numpy as np
import pytest

from gallium_b200 import GalliumError, _lib, paged

from test_gpu_paged import Case

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


def _attention_with_workspace(batch, c, out, words):
    """paged.attention into out over a workspace whose every 32-bit word is `words`."""
    torch = _torch()
    batch._set_pool(c.k, c.v)
    lib, d = _lib.load_library(), batch._desc
    n = ctypes.c_int64()
    _lib.check(lib.gb_paged_attention_workspace(batch._ref, c.heads, ctypes.byref(n)))
    ws = torch.full((n.value // 4,), words, dtype=torch.int32, device="cuda")
    a = _lib.AttnArgs()
    a.struct_size = ctypes.sizeof(a)
    a.n_heads, a.out_dtype, a.scale = c.heads, d.dtype, c.dim ** -0.5
    a.q_dev, a.k_pool_dev, a.v_pool_dev, a.out_dev = (t.data_ptr() for t in (c.q, c.k, c.v, out))
    a.q_row_stride, a.q_head_stride, _ = c.q.stride()
    a.out_row_stride, a.out_head_stride, _ = out.stride()
    a.workspace_dev, a.workspace_bytes = ws.data_ptr(), n.value
    _lib.check(lib.gb_paged_attention(batch._ref, ctypes.byref(a), torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("n_seqs", [128, 300])
@pytest.mark.parametrize("rows,lens", [(62, (64, 64)), (2, (64, 320))])
def test_sequences_that_share_rows_join_nothing_that_was_not_written(rows, lens, n_seqs):
    """q_start goes back, so that every second sequence holds the same rows: more items
    than CTAs, the last of them split (chunks), or a pair cut at the last CTA (single
    tokens).  Only rows of the sequences are written, whatever the workspace held (words
    of 1 are a group of row 1)."""
    torch = _torch()
    c = Case([(rows, 64)], heads=64, kvh=8, seed=1, spare_rows=3)
    c.starts = np.array([2, rows + 2] * (n_seqs // 2) + [2], np.int32)  # rows 0, 1 and the last are of none
    kv = np.array([lens[0], 0, lens[1], 0] * (n_seqs // 4), np.int32)
    if rows > 2:
        kv[n_seqs - 2] = 8192
    table = np.full((n_seqs, 512), c.table_np[0, 0], np.int32)  # a live page for every position
    batch = paged.PagedBatch(torch.from_numpy(c.starts).cuda(), torch.from_numpy(kv).cuda(),
                             torch.from_numpy(table).cuda(), page_size=16, total_q=c.total, max_q_len=rows,
                             max_kv_len=int(kv.max()))
    out = torch.full_like(c.q, 7.0)
    _attention_with_workspace(batch, c, out, 1)
    with pytest.raises(GalliumError, match="bounds"):
        batch.check()
    assert (out[:2] == 7.0).all() and (out[rows + 2:] == 7.0).all()
    # the same lengths without the shared rows, on the same workspace pattern
    ok = Case([(rows, 64), (rows, 3000)], heads=64, kvh=8, seed=2)
    out = torch.full_like(ok.q, 7.0)
    batch = ok.batch()
    _attention_with_workspace(batch, ok, out, 1)
    batch.check()
    assert torch.equal(out, paged.attention(ok.batch(), ok.q, ok.k, ok.v))
