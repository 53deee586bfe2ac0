"""The attention of paged caches where its inputs are at their worst: device arrays
that contradict themselves, values that are not finite, rows beside rows.  Batches
and tolerances are those of test_gpu_paged.py."""
import ctypes

import numpy as np
import pytest

from gallium_b200 import GalliumError, _lib, paged

from test_gpu_paged import SMALL, Case, U

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


# -- values that are not finite ------------------------------------------------------
# (lengths, row of the batch whose scores are all NaN, and whether one key makes them so)
NAN_LENS = {
    "decode": [(1, 40), (1, 17)],                # the 17th key is alone with one of the decoding kernel's warps
    "decode split": [(1, 40), (1, 6000)],
    "two tokens": [(1, 40), (2, 17)],
    "tile": [(1, 40), (40, 90)],
    "tile split": [(1, 40), (40, 9000)],
    "tile window": [(1, 40), (200, 300)],
}


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("heads,kvh,dim", [(8, 2, 64), (8, 2, 128), (6, 3, 128), (4, 2, 256)])
@pytest.mark.parametrize("lens", list(NAN_LENS))
def test_nan_reaches_the_rows_that_see_it(lens, heads, kvh, dim, sinks):
    """A query, or the last key of a sequence, holds NaN: what sees it is NaN, whichever
    kernel and however many parts worked on it; everything else keeps its bits."""
    torch = _torch()
    window = 64 if "window" in lens else 0
    c = Case(NAN_LENS[lens], heads=heads, kvh=kvh, dim=dim, seed=41)
    kw = dict(window=window, sinks=torch.linspace(-1, 1, heads).cuda() if sinks else None)
    clean = paged.attention(c.batch(), c.q, c.k, c.v, **kw)
    assert torch.isfinite(clean).all()
    n, kv = c.lens[1]
    row = int(c.starts[1]) + n // 2
    q = c.q.clone()
    q[row, 1, 5] = float("nan")
    out = paged.attention(c.batch(), q, c.k, c.v, **kw)
    assert torch.isnan(out[row, 1]).all()
    out[row, 1] = clean[row, 1]
    assert torch.equal(out, clean)
    # the last key, which the last row alone sees; of one KV head
    c.k[c.table_np[1, (kv - 1) // c.page], (kv - 1) % c.page, 0, 7] = float("nan")
    out = paged.attention(c.batch(), c.q, c.k, c.v, **kw)
    last, group = int(c.starts[2]) - 1, heads // kvh
    assert torch.isnan(out[last, :group]).all()
    out[last, :group] = clean[last, :group]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 17)], [(3, 200)], [(60, 60)], [(30, 9000)]])
def test_all_keys_nan(lens, dim):
    """Every visible score is NaN: no row is taken for one that sees nothing."""
    torch = _torch()
    c = Case(lens, heads=4, kvh=1, dim=dim, seed=42)
    c.k[...] = float("nan")
    out = paged.attention(c.batch(), c.q, c.k, c.v)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("heads,kvh,dim", [(8, 2, 64), (8, 2, 128), (6, 3, 128), (4, 2, 256)])
def test_values_of_single_tokens_that_are_not_finite(heads, kvh, dim, value):
    """Rows of one decoding tile see different keys: a value that is not finite in the
    last position, or in one that the window has left behind for the later row, changes
    no bit of the rows that do not see it."""
    torch = _torch()
    for window in (0, 50):
        c = Case([(1, 33), (3, 121)], heads=heads, kvh=kvh, dim=dim, seed=43)
        wide = lambda v: paged.attention(c.batch(), c.q, c.k, v, window=window, out=torch.empty_like(c.q, dtype=torch.float32))  # noqa: E731
        clean = wide(c.v)
        for bad in [120, 119] + ([118 - 49] if window else []):
            v = c.v.clone()
            v[c.table_np[1, bad // c.page], bad % c.page, 0, 3] = value
            out = wide(v)
            for i, pos in enumerate((118, 119, 120)):
                if pos >= bad and (not window or pos - bad < window):
                    assert not torch.isfinite(out[1 + i, :heads // kvh, 3]).any()
                    out[1 + i, :heads // kvh, 3] = clean[1 + i, :heads // kvh, 3]
            assert torch.equal(out, clean), (window, bad)


# -- bad pages -----------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(200, 6000)], [(150, 400), (1, 900), (90, 2500)]])
def test_bad_pages_in_many_tiles_are_masked_where_they_are(lens, dim):
    """Pages outside the pool here and there among a chunk's keys, found by the producer
    while other warps work on earlier tiles: their keys alone are masked."""
    torch = _torch()
    c = Case(lens, heads=4, kvh=2, dim=dim, seed=45)
    r = np.random.default_rng(46)
    keep = []
    for b, (_, kv) in enumerate(lens):
        pages = -(-kv // c.page)
        gone = r.choice(pages, pages // 6, replace=False)
        keep.append(~np.isin(np.arange(kv) // c.page, gone))
        c.table_np[b, gone] = r.choice([-1, c.n_pages, 2 ** 31 - 1, -2 ** 31], len(gone))
    outs = []
    for _ in range(3):
        batch = c.batch()
        outs.append(paged.attention(batch, c.q, c.k, c.v))
        with pytest.raises(GalliumError, match="page"):
            batch.check()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    for b, (n, kv) in enumerate(lens):
        table = np.where(keep[b][np.arange(-(-kv // c.page)) * c.page], c.table_np[b, :-(-kv // c.page)], 0)
        pages = torch.from_numpy(table).long().cuda()
        K, V = (x[pages].reshape(-1, c.kvh, c.dim)[:kv].double() for x in (c.k, c.v))
        hidden = torch.arange(kv, device="cuda")[None] > torch.arange(kv - n, kv, device="cuda")[:, None]
        hidden = hidden | ~torch.from_numpy(keep[b]).cuda()
        K[~torch.from_numpy(keep[b]).cuda()] = 0
        V[~torch.from_numpy(keep[b]).cuda()] = 0
        for h in range(c.heads):
            q, k, v = c.q[c.starts[b]:c.starts[b] + n, h].double(), K[:, h // 2], V[:, h // 2]
            w = torch.softmax((q @ k.T * dim ** -0.5).masked_fill(hidden, -float("inf")), 1)
            e = (q.abs() @ k.abs().T).amax(1, keepdim=True) * dim ** -0.5 * (dim + 4) * U["f32"]
            tol = (w @ v.abs()) * (U[c.dtype] + 2 * (e + 2.0 ** -20) + kv * U["f32"]) + U[c.dtype] * (w @ v).abs()
            got = outs[0][c.starts[b]:c.starts[b] + n, h].double()
            assert ((got - w @ v).abs() <= tol + SMALL[U[c.dtype]]).all(), (b, h)


# -- rows beside rows ----------------------------------------------------------------
@pytest.mark.parametrize("heads,kvh,dim", [(8, 2, 64), (3, 1, 64), (5, 1, 128), (6, 2, 128), (14, 2, 256), (9, 1, 64)])
@pytest.mark.parametrize("lens", [[(2, 150), (1, 300)], [(20, 700), (25, 25)], [(150, 2000), (30, 300), (1, 9)]])
def test_a_row_keeps_its_bits_whatever_its_neighbours_hold(lens, heads, kvh, dim):
    """Larger queries in other rows, of its own tile too, and what earlier work left in
    shared memory have no part in a row's rounding."""
    torch = _torch()
    c = Case(lens, heads=heads, kvh=kvh, dim=dim, dtype="f16", seed=44)
    want = paged.attention(c.batch(), c.q, c.k, c.v)
    other = c.batch()
    for keep in (0, c.total // 2, c.total - 1):
        q = c.q * 60
        q[keep] = c.q[keep]
        for _ in range(3):
            out = paged.attention(other, q, c.k, c.v)
            assert torch.equal(out[keep], want[keep])
            assert torch.equal(paged.attention(c.batch(), c.q, c.k, c.v), want)
