"""gb_paged_rope_append, gb_paged_attention and gb_paged_copy against plain
float64 restatements of their definitions: ragged batches, page sizes, head
layouts, windows, sinks, rows that see nothing, garbage in every place that a
row does not see, strides, another stream, graph replay.

Tolerances are counted in roundings (u = half a step of the type: bf16 2^-8,
f16 2^-11, f32 2^-24).  Attention: the output's rounding u |o|; each
probability's rounding to the pool's type, u sum p |v|; and the f32 scores, of
absolute error e = scale sum |q k| (dim + 4) 2^-24, with the exponential's own
2^-21, each of which moves every p by a relative amount: 2 (e + 2^-20) sum p |v|
(numerator and denominator), p normalised; f32 sums of n terms add n 2^-24.
Rotation: u |y| + (|x1 cos| + |x2 sin|) (dim + 32) 2^-24 for the norm's sum and
the few f32 operations after it."""
import math

import numpy as np
import pytest

from gallium_b200 import GalliumError, _lib, paged

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
# Below the smallest normal number (f16 2^-14, the others 2^-126) the spacing stays
# (2^-24, 2^-133, 2^-149), so a rounding is off by half of it whatever the value.
SMALL = {2.0 ** -8: 2.0 ** -134, 2.0 ** -11: 2.0 ** -25, 2.0 ** -24: 2.0 ** -150}


def _torch():
    import torch

    return torch


def _t(name):
    torch = _torch()
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


class Case:
    """A ragged batch with pages in random order and random pools."""

    def __init__(self, lens, *, heads=8, kvh=2, dim=64, page=16, dtype="bf16", seed=0, spare_rows=0,
                 head_major=False, poison=True):
        torch = _torch()
        self.lens, self.heads, self.kvh, self.dim, self.page, self.dtype = lens, heads, kvh, dim, page, dtype
        g = self.g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        t = _t(dtype)
        need = [-(-kv // page) for _, kv in lens]
        self.n_pages = sum(need) + 2
        order = torch.randperm(self.n_pages, generator=g, device="cuda").tolist()
        width = max(need + [1]) + 1
        table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table_np = table
        self.total = sum(q for q, _ in lens) + spare_rows
        shape = (self.n_pages, kvh, page, dim) if head_major else (self.n_pages, page, kvh, dim)
        self.k, self.v = (torch.empty(shape, dtype=t, device="cuda").normal_(generator=g) for _ in range(2))
        if head_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        if poison:  # whatever no sequence holds
            live = torch.zeros(self.n_pages, page, dtype=torch.bool, device="cuda")
            for b, (_, kv) in enumerate(lens):
                for p in range(need[b]):
                    live[table[b, p], :min(page, kv - p * page)] = True
            for pool in (self.k, self.v):
                pool[~live] = float("nan")
        self.q = torch.empty(self.total, heads, dim, dtype=t, device="cuda").normal_(generator=g)
        self.starts = np.concatenate([[0], np.cumsum([q for q, _ in lens])]).astype(np.int32)

    def batch(self, **kw):
        torch = _torch()
        args = dict(page_size=self.page, total_q=self.total, max_q_len=max(q for q, _ in self.lens),
                    max_kv_len=max(kv for _, kv in self.lens))
        args.update(kw)
        return paged.PagedBatch(torch.from_numpy(self.starts).cuda(),
                                torch.tensor([kv for _, kv in self.lens], dtype=torch.int32).cuda(),
                                torch.from_numpy(self.table_np).cuda(), **args)

    def keys(self, b, pool):
        """Sequence b's cached rows [kv, kvh, dim] in float64."""
        kv = self.lens[b][1]
        pages = self.table_np[b, :-(-kv // self.page)]
        assert ((pages >= 0) & (pages < self.n_pages)).all()  # on the host, before torch indexes with them
        x = pool[_torch().from_numpy(pages).long().cuda()].double().cpu().numpy()
        return x.reshape(-1, self.kvh, self.dim)[:kv]

    def attention(self, window=0, sinks=None, scale=None):
        """(out, tolerance without the output's own rounding) in float64."""
        scale = self.dim ** -0.5 if scale is None else scale
        q = self.q.double().cpu().numpy()
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        for b, (n, kv) in enumerate(self.lens):
            K, V = self.keys(b, self.k), self.keys(b, self.v)
            for i in range(n):
                p = kv - n + i
                lo = max(0, p - window + 1) if window else 0
                if p < 0:
                    continue
                r = self.starts[b] + i
                for h in range(self.heads):
                    k, v = K[lo:p + 1, h * self.kvh // self.heads], V[lo:p + 1, h * self.kvh // self.heads]
                    s = k @ q[r, h] * scale
                    e = (np.abs(k) @ np.abs(q[r, h])).max() * abs(scale) * (self.dim + 4) * U["f32"]
                    m = s.max() if sinks is None else max(s.max(), sinks[h])
                    w = np.exp(s - m)
                    w = w / (w.sum() + (0 if sinks is None else math.exp(sinks[h] - m)))
                    out[r, h] = w @ v
                    tol[r, h] = (w @ np.abs(v)) * (U[self.dtype] + 2 * (e + 2.0 ** -20) + len(s) * U["f32"])
        return out, tol


def _check_large(c, window=0, sinks=None, batch=None):
    """The same check as _check_attention with the float64 reference on the GPU,
    for batches that the row by row one is too slow for."""
    torch = _torch()
    s = None if sinks is None else torch.tensor(sinks, dtype=torch.float32).cuda()
    batch = batch or c.batch()
    out = paged.attention(batch, c.q, c.k, c.v, sinks=s, window=window)
    batch.check()
    for b, (n, kv) in enumerate(c.lens):
        if not n:
            continue
        pages = torch.from_numpy(c.table_np[b, :-(-kv // c.page)]).long().cuda()
        K, V = (x[pages].reshape(-1, c.kvh, c.dim)[:kv].double() for x in (c.k, c.v))
        q = c.q[c.starts[b]:c.starts[b] + n].double()
        pos = torch.arange(kv - n, kv, device="cuda")[:, None]
        key = torch.arange(kv, device="cuda")[None]
        hidden = (key > pos) | ((pos - key >= window) if window else False)
        for h in range(c.heads):
            k, v = K[:, h * c.kvh // c.heads], V[:, h * c.kvh // c.heads]
            a = (q[:, h] @ k.T * c.dim ** -0.5).masked_fill(hidden, -math.inf)
            e = (q[:, h].abs() @ k.abs().T).masked_fill(hidden, 0).amax(1, keepdim=True) * c.dim ** -0.5
            if s is not None:
                a = torch.cat([a, s[h].double().expand(n, 1)], 1)
            w = torch.softmax(a, 1)[:, :kv]
            want, A = w @ v, w @ v.abs()
            tol = A * (U[c.dtype] + 2 * (e * (c.dim + 4) * U["f32"] + 2.0 ** -20) + kv * U["f32"]) + U[c.dtype] * want.abs()
            got = out[c.starts[b]:c.starts[b] + n, h].double()
            bad = (got - want).abs() - tol - SMALL[U[c.dtype]]
            assert torch.isfinite(got).all() and bad.max() <= 0, (b, h, float(bad.max()))
    return out


def _close(got, want, tol, u):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    err = np.abs(got - want) - (tol + u * np.abs(want) + SMALL[u])
    assert (err <= 1e-30).all(), (float(err.max()), np.unravel_index(err.argmax(), err.shape))


def _check_attention(c, window=0, sinks=None, scale=None, f32_out=False, batch=None):
    torch = _torch()
    s = None if sinks is None else torch.tensor(sinks, dtype=torch.float32).cuda()
    out = torch.full(c.q.shape, 7.0, dtype=torch.float32 if f32_out else c.q.dtype, device="cuda")
    batch = batch or c.batch()
    paged.attention(batch, c.q, c.k, c.v, sinks=s, window=window, scale=scale, out=out)
    batch.check()
    used = c.starts[-1]
    want, tol = c.attention(window, None if sinks is None else s.double().cpu().numpy(), scale)
    _close(out[:used], want[:used], tol[:used], U["f32" if f32_out else c.dtype])
    assert (out[used:] == 7.0).all()  # rows of no sequence
    return out


# -- attention -----------------------------------------------------------------
LENS = {
    "one": [(1, 1)],
    "decode": [(1, 1), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 300)],
    "decode long": [(1, 3001)],
    "two tokens": [(2, 2), (2, 130), (2, 65)],
    "chunks": [(37, 37), (5, 150), (64, 64), (1, 129), (130, 300)],
    "idle": [(0, 0), (3, 20), (0, 50), (1, 7), (0, 0)],
    "long chunk": [(17, 2000)],
}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens", list(LENS))
def test_attention_lengths(lens, dtype):
    _check_attention(Case(LENS[lens], dtype=dtype, seed=1, spare_rows=3))


@pytest.mark.parametrize("dim,heads,kvh", [(64, 16, 2), (128, 8, 2), (256, 4, 2)])
@pytest.mark.parametrize("window", [0, 200])
def test_attention_long_chunks(dim, heads, kvh, window):
    """Prompts of many tiles (every key tile count, several waves of CTAs), with
    and without cached keys, beside decoding sequences."""
    lens = [(2048, 2048), (1, 3000), (777, 1500), (601, 601), (1, 5), (64, 4000)]
    _check_large(Case(lens, heads=heads, kvh=kvh, dim=dim, seed=21, page=64), window=window,
                 sinks=np.linspace(-2, 2, heads))


@pytest.mark.parametrize("dim,heads,kvh,dtype", [(64, 8, 1, "bf16"), (128, 12, 4, "f16"), (256, 2, 2, "bf16")])
def test_attention_many_sequences(dim, heads, kvh, dtype):
    """More sequences than a warp holds, of very different lengths; some idle."""
    r = np.random.default_rng(22)
    lens = [(1, int(n)) for n in np.exp(r.uniform(0, np.log(3000), 300))]
    lens[7] = lens[150] = lens[299] = (0, 40)
    lens[40] = (2, 2)
    for extra in ([], [(300, 900), (40, 40)]):
        _check_large(Case(lens + extra, heads=heads, kvh=kvh, dim=dim, dtype=dtype, seed=23))


@pytest.mark.parametrize("n", [1, 2, 3, 127, 128, 129, 256])
def test_attention_equal_sequences(n):
    """Shares that end with a pair, and shares that cut every pair."""
    for kv in (64, 129, 1000):
        _check_large(Case([(1, kv)] * n, heads=8, kvh=4, seed=24 + n), sinks=[0.5] * 8)


@pytest.mark.parametrize("heads,kvh,dim", [(1, 1, 64), (3, 1, 128), (16, 1, 64), (10, 2, 64), (7, 7, 128), (12, 4, 256),
                                           (64, 8, 64), (24, 2, 128), (14, 2, 256)])
def test_attention_head_layouts(heads, kvh, dim):
    _check_attention(Case([(1, 40), (20, 90), (1, 700), (150, 200)], heads=heads, kvh=kvh, dim=dim, seed=2))


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("head_major", [False, True])
def test_attention_page_sizes_and_layouts(page, head_major):
    _check_attention(Case([(1, 200), (33, 260), (140, 140)], page=page, head_major=head_major, seed=3))


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 1000])
def test_attention_windows(window):
    sinks = np.linspace(-3, 3, 8)
    _check_attention(Case([(1, 333), (1, 64), (50, 130), (160, 300)], seed=4), window=window, sinks=sinks)


def test_pages_behind_the_window_may_be_gone():
    for lens in ([(1, 500), (20, 300)], [(150, 500)]):
        c = Case(lens, seed=5)
        want, tol = c.attention(window=100)
        for b, (n, kv) in enumerate(c.lens):
            first = max(0, kv - n - 100 + 1) // c.page
            gone = c.table_np[b, :first].copy()
            c.table_np[b, :first] = -1
            for pool in (c.k, c.v):
                pool[_torch().from_numpy(gone).long().cuda()] = float("inf")
        batch = c.batch()
        out = paged.attention(batch, c.q, c.k, c.v, window=100)
        batch.check()
        _close(out, want, tol, U[c.dtype])


@pytest.mark.parametrize("sink", [-float("inf"), -50.0, 0.0, 40.0])
def test_attention_sinks(sink):
    _check_attention(Case([(1, 50), (9, 9), (1, 2000), (130, 400)], seed=6), sinks=[sink] * 8)


def test_rows_before_position_zero_see_nothing():
    """kv_len below q_len: the first rows sit before the cache and give zeros."""
    for sinks in (None, [0.5] * 8):
        for n in (6, 150):
            c = Case([(n, n - 4), (n, 0), (2, 30)], seed=7)
            out = _check_attention(c, sinks=sinks)
            assert (out[:4] == 0).all() and (out[n:2 * n] == 0).all()


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_later_rows_have_no_part_in_earlier_ones(value):
    """K and V of one new token are not finite: rows before it are untouched,
    with a window also the rows that no longer see it; rows that see it are
    not finite."""
    torch = _torch()
    for lens, n, window in (([(2, 20), (8, 40)], 8, 0), ([(200, 300)], 200, 0), ([(200, 300)], 200, 32)):
        c = Case(lens, seed=8)
        clean = paged.attention(c.batch(), c.q, c.k, c.v, window=window)
        b = len(lens) - 1
        kv = lens[b][1]
        bad = kv - n // 2  # a position inside the chunk
        page, slot = c.table_np[b, bad // c.page], bad % c.page
        c.v[page, slot] = value
        out = paged.attention(c.batch(), c.q, c.k, c.v, window=window)
        pos = torch.arange(kv - n, kv)
        sees = (pos >= bad) & ((pos - bad < window) if window else True)
        rows = out[c.starts[b]:]
        assert torch.equal(rows[~sees], clean[c.starts[b]:][~sees])
        assert not torch.isfinite(rows[sees]).any()
        assert torch.equal(out[:c.starts[b]], clean[:c.starts[b]])
        c.k[page, slot] = value
        out = paged.attention(c.batch(), c.q, c.k, c.v, window=window)[c.starts[b]:]
        assert torch.equal(out[~sees], clean[c.starts[b]:][~sees])


# Rows behind the last sequence make a batch one of many tiles (more than 592 of 128
# rows), whose chunks at head_dim 64 run four to an SM.
MANY = dict(heads=16, kvh=2, dim=64, spare_rows=4800)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("window", [0, 1, 64, 100])
def test_attention_of_many_tiles(window, dtype):
    c = Case([(160, 300), (1, 333), (50, 130), (20, 16), (0, 40), (7, 0), (129, 129)], dtype=dtype, seed=31, **MANY)
    _check_attention(c, window=window, sinks=np.linspace(-2, 2, 16))


@pytest.mark.parametrize("window", [0, 128])
def test_attention_of_many_tiles_long(window):
    lens = [(2048, 2048), (1, 3000), (777, 1500), (601, 8000), (1, 5), (64, 4000)]
    c = Case(lens, heads=64, kvh=8, dim=64, seed=32, page=64)
    sinks = np.linspace(-2, 2, 64)
    first = _check_large(c, window=window, sinks=sinks)
    s = _torch().tensor(sinks, dtype=_torch().float32).cuda()
    for _ in range(3):  # the same result every time
        assert _torch().equal(paged.attention(c.batch(), c.q, c.k, c.v, window=window, sinks=s), first)


@pytest.mark.parametrize("window", [0, 500])
def test_attention_of_many_tiles_split_and_of_many_sequences(window):
    _check_large(Case([(48, 8000), (1, 7000), (33, 3333)], seed=37, page=32, **MANY), window=window,
                 sinks=np.linspace(-2, 2, 16))
    r = np.random.default_rng(38)
    lens = [(int(q), int(q + k)) for q, k in zip(np.exp(r.uniform(0, np.log(120), 260)), np.exp(r.uniform(0, np.log(1500), 260)))]
    lens[3] = lens[200] = (0, 30)
    _check_large(Case(lens, seed=39, **MANY), window=window)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_many_tiles_keep_values_that_are_not_finite_to_the_rows_that_see_them(value):
    torch = _torch()
    for window in (0, 32):
        c = Case([(200, 300), (40, 40)], seed=33, **MANY)
        clean = paged.attention(c.batch(), c.q, c.k, c.v, window=window)
        bad = 300 - 100
        c.v[c.table_np[0, bad // c.page], bad % c.page] = value
        out = paged.attention(c.batch(), c.q, c.k, c.v, window=window)
        pos = torch.arange(100, 300)
        sees = torch.zeros(240, dtype=torch.bool)
        sees[:200] = (pos >= bad) & ((pos - bad < window) if window else True)
        assert torch.equal(out[:240][~sees], clean[:240][~sees])
        assert not torch.isfinite(out[:240][sees]).any()


def test_calls_on_two_streams_at_once():
    """Batches of few and of many tiles, of different head dims, in flight together."""
    torch = _torch()
    cases = [Case([(160, 900), (1, 700)], seed=34, **MANY), Case([(300, 300), (1, 5000)], heads=8, kvh=2, seed=35),
             Case([(260, 800), (1, 900)], heads=8, kvh=2, dim=128, seed=36)]
    batches = [c.batch() for c in cases]
    want = [paged.attention(b, c.q, c.k, c.v, out=torch.zeros_like(c.q)) for b, c in zip(batches, cases)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(10):
        for i, (b, c) in enumerate(zip(batches, cases)):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged.attention(b, c.q, c.k, c.v, out=torch.zeros_like(c.q)))
    torch.cuda.synchronize()
    for i, b in enumerate(batches):
        b.check()
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_large_scores_and_masks_of_the_lowest_value():
    """Scores of +-10^4 (one key takes all), and keys whose scores are all the
    type's lowest value."""
    c = Case([(1, 100), (40, 80), (150, 150)], seed=9)
    c.q *= 100
    _check_attention(c, scale=12.5)
    c = Case([(1, 100), (140, 150)], seed=9)
    low = _torch().finfo(c.k.dtype).min
    c.k[:] = 0
    c.k[..., 0] = low
    c.q[:] = 0
    c.q[..., 0] = 1
    _check_attention(c, scale=1.0)


def test_attention_f32_output_and_strides():
    torch = _torch()
    c = Case([(3, 30), (1, 200), (150, 170)], seed=10)
    _check_attention(c, f32_out=True)
    # q inside a projection's rows, out with a padded row
    wide = torch.zeros(c.total, 8 * 64 + 2 * 2 * 64, dtype=c.q.dtype, device="cuda")
    wide[:, :512] = c.q.reshape(c.total, -1)
    plain = paged.attention(c.batch(), c.q, c.k, c.v)
    room = torch.full((c.total, 11, 64), 3.0, dtype=c.q.dtype, device="cuda")
    paged.attention(c.batch(), wide[:, :512].view(c.total, 8, 64), c.k, c.v, out=room[:, 2:10])
    assert torch.equal(room[:, 2:10], plain)
    assert (room[:, :2] == 3).all() and (room[:, 10:] == 3).all()


def test_attention_is_deterministic_and_runs_on_another_stream():
    torch = _torch()
    c = Case([(1, 3000), (1, 10), (200, 900), (1, 1500)], seed=11)
    batch = c.batch()
    first = paged.attention(batch, c.q, c.k, c.v)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(5):
            assert torch.equal(paged.attention(batch, c.q, c.k, c.v), first)
    s.synchronize()


def test_bad_device_arrays_are_flagged_and_contained():
    torch = _torch()
    c = Case([(1, 100), (1, 40), (140, 200)], seed=12)
    want, tol = c.attention()
    live = np.r_[0:32, 48:100]
    K, V = (c.keys(0, pool)[live] for pool in (c.k, c.v))
    c.table_np[0, 2] = c.n_pages  # a needed page that is not in the pool
    batch = c.batch()
    out = paged.attention(batch, c.q, c.k, c.v)
    with pytest.raises(GalliumError) as e:
        batch.check()
    assert e.value.status == _lib.GB_ERR_INVALID_ARG and "page" in str(e.value)
    batch.check()  # cleared
    _close(out[1:], want[1:], tol[1:], U[c.dtype])
    # its keys count as masked
    for h in range(8):
        s = K[:, h // 4] @ c.q[0, h].double().cpu().numpy() / 8
        w = np.exp(s - s.max())
        w /= w.sum()
        t = (w @ np.abs(V[:, h // 4])) * 1.01 * U["bf16"] + U["bf16"] * np.abs(w @ V[:, h // 4]) + 1e-4
        assert (np.abs(out[0, h].double().cpu().numpy() - w @ V[:, h // 4]) <= t).all()
    c = Case([(1, 100), (1, 40)], seed=12)
    for name, kw in (("long", dict(max_kv_len=50)),):
        batch = c.batch(**kw)
        paged.attention(batch, c.q, c.k, c.v)
        with pytest.raises(GalliumError, match="bounds"):
            batch.check()
    c.starts = np.array([0, 5, 2], np.int32)
    batch = c.batch()
    paged.attention(batch, c.q, c.k, c.v)
    torch.cuda.synchronize()
    with pytest.raises(GalliumError, match="bounds"):
        batch.check()


# -- norm, rotation, append ------------------------------------------------------
def _tables(n, rot):
    torch = _torch()
    f = 10000.0 ** (-np.arange(rot // 2) * 2.0 / rot)
    a = np.arange(n)[:, None] * f
    return (torch.from_numpy(x.astype(np.float32)).cuda() for x in (np.cos(a), np.sin(a)))


def _turn(x, w, eps, pos, cos, sin, rot):
    """Norm and rotation of x [n, heads, dim] in float64, and the tolerance's base."""
    x = np.asarray(x, np.float64)
    dim = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w
    if rot == 0:
        return x, np.abs(x) * (dim + 32) * U["f32"]
    h = rot // 2
    c, s = cos[pos][:, None], sin[pos][:, None]
    x1, x2, rest = x[..., :h], x[..., h:rot], x[..., rot:]
    y = np.concatenate([x1 * c - x2 * s, x1 * s + x2 * c, rest], -1)
    base = np.concatenate([abs(x1 * c) + abs(x2 * s), abs(x1 * s) + abs(x2 * c), abs(rest)], -1)
    return y, base * (dim + 32) * U["f32"]


@pytest.mark.parametrize("heads,kvh,dim,rot,norm,din,dtype", [
    (8, 2, 64, 64, False, "bf16", "bf16"), (8, 2, 64, 32, True, "f16", "f16"), (5, 1, 128, 128, True, "bf16", "bf16"),
    (4, 4, 256, 64, True, "f32", "bf16"), (64, 8, 64, 64, False, "f32", "f16"), (3, 3, 128, 0, True, "f16", "f16"),
    (2, 1, 256, 256, False, "bf16", "f16"), (16, 8, 128, 16, True, "bf16", "bf16"), (1, 1, 64, 0, False, "f32", "bf16"),
])
@pytest.mark.parametrize("lens", ["one", "decode", "idle", "chunks", "many"])
def test_rope_append(lens, heads, kvh, dim, rot, norm, din, dtype):
    torch = _torch()
    lens = LENS[lens] if lens != "many" else [(300, 310), (1, 40), (700, 700), (0, 9), (1000, 1100)]
    c = Case(lens, heads=heads, kvh=kvh, dim=dim, dtype=dtype, seed=13, spare_rows=2, head_major=dim == 128)
    n = c.total
    x = torch.empty(n, heads + 2 * kvh, dim, dtype=_t(din), device="cuda").normal_(0, 2, generator=c.g)
    q, k, v = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]
    w = [1 + 0.3 * torch.randn(dim, generator=c.g, device="cuda") for _ in range(2)] if norm else [None, None]
    cos, sin = _tables(1200, rot) if rot else (None, None)
    before = [p.clone() for p in (c.k, c.v)]
    q_out = torch.full((n, heads, dim), 9.0, dtype=_t(dtype), device="cuda")
    batch = c.batch()
    got = paged.rope_append(batch, q, k, v, c.k, c.v, cos, sin, q_norm=w[0], k_norm=w[1], eps=1e-5, q_out=q_out)
    batch.check()
    assert got is q_out
    used = c.starts[-1]
    assert (q_out[used:] == 9.0).all()
    pos = np.concatenate([np.arange(kv - m, kv) for m, kv in lens]).astype(int)
    cn, sn = (t.double().cpu().numpy() if rot else None for t in (cos, sin))
    xs = x[:used].double().cpu().numpy()
    wn = [t.double().cpu().numpy() if norm else None for t in w]
    want, tol = _turn(xs[:, :heads], wn[0], 1e-5, pos, cn, sn, rot)
    _close(q_out[:used], want, tol, U[dtype])
    kw, ktol = _turn(xs[:, heads:heads + kvh], wn[1], 1e-5, pos, cn, sn, rot)
    written = torch.zeros(c.n_pages, c.page, dtype=torch.bool, device="cuda")
    at = 0
    for b, (m, kv) in enumerate(lens):
        p = np.arange(kv - m, kv)
        pages, slots = c.table_np[b, p // c.page], p % c.page
        ix = torch.from_numpy(pages).long().cuda(), torch.from_numpy(slots).long().cuda()
        written[ix] = True
        _close(c.k[ix], kw[at:at + m], ktol[at:at + m], U[dtype])
        assert torch.equal(c.v[ix], v[at:at + m].to(_t(dtype)))
        at += m
    for pool, old in zip((c.k, c.v), before):  # every other slot as it was, NaN included
        assert torch.equal(pool[~written].view(torch.int16), old[~written].view(torch.int16))


def test_rope_append_in_place_equals_out_of_place():
    torch = _torch()
    c = Case([(40, 50), (1, 99)], seed=14)
    cos, sin = _tables(128, 64)
    k = torch.randn(c.total, 2, 64, device="cuda").to(c.q.dtype)
    want = paged.rope_append(c.batch(), c.q, k, k, c.k, c.v, cos, sin)
    assert paged.rope_append(c.batch(), c.q, k, k, c.k, c.v, cos, sin, q_out=c.q) is c.q
    assert torch.equal(c.q, want)


def test_rope_append_drops_bad_rows_and_pages():
    torch = _torch()
    c = Case([(4, 2), (3, 40), (2, 20)], seed=15, poison=False)  # rows before position 0
    cos, sin = _tables(39, 64)  # position 39 is past the tables
    c.table_np[2, 1] = -1  # the page of positions 18 and 19
    before = [p.clone() for p in (c.k, c.v)]
    q_out = torch.full_like(c.q, 9.0)
    k = torch.ones(c.total, 2, 64, device="cuda", dtype=c.q.dtype)
    batch = c.batch()
    paged.rope_append(batch, c.q, k, k, c.k, c.v, cos, sin, q_out=q_out)
    with pytest.raises(GalliumError) as e:
        batch.check()
    assert "page" in str(e.value) and "position" in str(e.value)
    assert (q_out[:2] == 9).all() and (q_out[6] == 9).all() and not (q_out[2:6] == 9).all()
    changed = (c.v != before[1]).flatten(2).any(-1).nonzero().tolist()
    want = [[int(c.table_np[0, 0]), 0], [int(c.table_np[0, 0]), 1], [int(c.table_np[1, 37 // 16]), 37 % 16],
            [int(c.table_np[1, 38 // 16]), 38 % 16]]
    assert sorted(changed) == sorted(want)


def test_python_refuses_mismatched_tensors():
    torch = _torch()
    c = Case([(1, 20)], seed=16)
    b = c.batch()
    for call in (lambda: paged.attention(b, c.q.float(), c.k, c.v), lambda: paged.attention(b, c.q[:, :, :32], c.k, c.v),
                 lambda: paged.attention(b, c.q, c.k, c.v.half()), lambda: paged.attention(b, c.q, c.k[:, :8], c.v[:, :8]),
                 lambda: paged.attention(b, c.q, c.k, c.v, sinks=torch.zeros(3).cuda()),
                 lambda: paged.attention(b, c.q.cpu(), c.k, c.v), lambda: paged.attention(b, c.q, c.k, c.v, out=c.q),
                 lambda: paged.rope_append(b, c.q, c.q, c.q, c.k, c.v),
                 lambda: paged.rope_append(b, c.q, c.q[:, :2], c.q[:, :2], c.k, c.v, cos=torch.zeros(30, 32).cuda()),
                 lambda: paged.copy_pages([c.k, c.v.float()], [0], [1]),
                 lambda: paged.copy_pages([c.k[:, :, :1]], [0], [1])):
        with pytest.raises(GalliumError):
            call()


# -- page copies -----------------------------------------------------------------
@pytest.mark.parametrize("shape,n", [((3, 9, 16, 2, 64), 4), ((2, 700, 8, 1, 64), 300), ((70, 12, 16, 2, 64), 5),
                                     ((2, 5, 128, 8, 128), 2), ((1, 5000, 8), 2400), ((2, 7, 24), 3)])
def test_copy_pages(shape, n):
    torch = _torch()
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    pools = torch.randint(-2 ** 15, 2 ** 15, shape, generator=g, device="cuda", dtype=torch.int16)
    order = torch.randperm(shape[1], generator=g, device="cuda").tolist()
    src, dst = [order[i // 2] for i in range(n)], order[shape[1] - n:]  # each source twice
    want = pools.clone()
    want[:, dst] = want[:, src]
    paged.copy_pages(pools, src, dst)
    assert torch.equal(pools, want)
    listed = [p.clone() for p in pools]
    paged.copy_pages(listed, dst[:1], src[:1])
    for p, w in zip(listed, want):
        w = w.clone()
        w[src[0]] = w[dst[0]]
        assert torch.equal(p, w)


def test_copy_pages_between_strided_and_head_major_pages():
    torch = _torch()
    wide = torch.randn(6, 3, 2, 16, 64, device="cuda", dtype=torch.float16)
    pool = wide[:, 1].transpose(1, 2)  # [page][slot][head][dim] of a page-strided, head-major pool
    want = wide.clone()
    want[4, 1] = want[2, 1]
    paged.copy_pages([pool], [2], [4])
    assert torch.equal(wide, want)
    paged.copy_pages([pool], [], [])


# -- as they are used ------------------------------------------------------------
def test_a_serving_loop_with_forks_and_a_compaction():
    """Prefill in chunks, decode, a fork, a window's end, a compaction: the
    cached path gives what attention over the whole history gives."""
    torch = _torch()
    heads, kvh, dim, page = 8, 2, 64, 16
    pool = paged.PagePool(64, page)
    kp, vp = (torch.full((64, page, kvh, dim), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cos, sin = _tables(512, dim)
    g = torch.Generator(device="cuda")
    g.manual_seed(17)
    history = {}

    def step(new):
        """new: {sequence: tokens}; returns the outputs, checked against the histories."""
        src, dst = [], []
        for s, n in new.items():
            a, b = pool.extend(s, n)
            src += a
            dst += b
        paged.copy_pages([kp, vp], src, dst)
        seqs, ns = list(new), list(new.values())
        total = sum(ns)
        x = torch.empty(total, heads + 2 * kvh, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        kv = [pool.length(s) for s in seqs]
        batch = paged.PagedBatch(torch.tensor(np.concatenate([[0], np.cumsum(ns)]), dtype=torch.int32).cuda(),
                                 torch.tensor(kv, dtype=torch.int32).cuda(),
                                 torch.from_numpy(pool.table(seqs)).cuda(), page_size=page, total_q=total,
                                 max_q_len=max(ns), max_kv_len=max(kv))
        q = paged.rope_append(batch, x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:], kp, vp, cos, sin)
        out = paged.attention(batch, q, kp, vp)
        batch.check()
        at = 0
        for s, n in new.items():
            h = history.setdefault(s, [])
            for i in range(at, at + n):
                h.append((x[i, heads:heads + kvh].double().cpu().numpy(), x[i, heads + kvh:].double().cpu().numpy()))
            K = np.stack([a for a, _ in h])
            V = np.stack([b for _, b in h])
            cn, sn = cos.double().cpu().numpy(), sin.double().cpu().numpy()
            K, _ = _turn(K, None, 0, np.arange(len(h)), cn, sn, dim)
            for i in range(n):
                p = len(h) - n + i
                qq = q[at + i].double().cpu().numpy()
                for hd in range(heads):
                    sc = K[:p + 1, hd // 4] @ qq[hd] / 8
                    w = np.exp(sc - sc.max())
                    w /= w.sum()
                    A = w @ np.abs(V[:p + 1, hd // 4])
                    # keys are rounded once (u |k|), which moves a score by u sum |q k| / 8
                    e = U["bf16"] * (np.abs(K[:p + 1, hd // 4]) @ np.abs(qq[hd])).max() / 8
                    err = np.abs(out[at + i, hd].double().cpu().numpy() - w @ V[:p + 1, hd // 4])
                    assert (err <= A * (2 * e + 2 * U["bf16"] + 1e-4) + U["bf16"] * A).all()
            at += n

    a, b = pool.add(), pool.add()
    step({a: 37, b: 5})
    step({a: 20, b: 1})
    c = pool.fork(a)
    history[c] = list(history[a])
    step({a: 1, b: 1, c: 1})
    for _ in range(3):
        step({c: 1, a: 1})
    pool.free(b)
    del history[b]
    src, dst = pool.compact()
    paged.copy_pages([kp, vp], src, dst)
    assert src
    step({a: 1, c: 2})
    pool.truncate(c, 40)
    del history[c][40:]
    step({a: 1, c: 30})


def test_a_captured_decode_step_follows_its_device_lengths():
    """rope_append and attention captured once, replayed while kv_len, the
    page table and the inputs change in place."""
    torch = _torch()
    c = Case([(1, 200), (1, 200), (1, 200)], seed=18)
    cos, sin = _tables(256, 64)
    x = torch.randn(3, 12, 64, device="cuda").to(c.q.dtype)
    kv = torch.tensor([5, 60, 100], dtype=torch.int32).cuda()
    batch = paged.PagedBatch(torch.arange(4, dtype=torch.int32).cuda(), kv, torch.from_numpy(c.table_np).cuda(),
                             page_size=16, total_q=3, max_q_len=1, max_kv_len=200)
    out = torch.empty_like(c.q)

    def go():
        q = paged.rope_append(batch, x[:, :8], x[:, 8:10], x[:, 10:], c.k, c.v, cos, sin)
        paged.attention(batch, q, c.k, c.v, out=out, sinks=None)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for step in range(20):
        kv.add_(3)
        x.normal_()
        graph.replay()
        got = out.clone()
        go()
        assert torch.equal(got, out), step
    batch.check()
