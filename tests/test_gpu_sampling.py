"""gb_sample against the definition in float64: tokens equal, log-probabilities
within a few f32 roundings of their size."""
import math

import numpy as np
import pytest

from gallium_b200 import GalliumError, sampling

pytestmark = pytest.mark.gpu


def _want(x, u, t=1.0, k=0, p=1.0, least=0.0):
    """(token, log-probability) of one row, from the definition."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1, -np.inf
    if not t > 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.exp(np.where(x == top, 0.0, (x - top) / t)))
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        s = w[order]
        before = np.concatenate([[0.0], np.cumsum(s)[:-1]])
        keep = before < p * s.sum()
        keep[0] = True
        order = order[keep]
    order = np.concatenate([order[:1], order[1:][w[order[1:]] >= least]])
    ids = np.sort(order)
    c = np.cumsum(w[ids])
    u = min(max(u, 0.0), 1 - 2.0 ** -24)
    i = min(int(np.searchsorted(c, u * c[-1], side="right")), len(ids) - 1)
    return int(ids[i]), math.log(w[ids[i]] / c[-1])


def _run(x, u, t=None, k=None, p=None, least=None, **kw):
    import torch

    def dev(v, d):
        return None if v is None else torch.tensor(np.asarray(v), dtype=d).cuda()

    tok, lp = sampling.sample(x, dev(u, torch.float32), temperature=dev(t, torch.float32), top_k=dev(k, torch.int32),
                              top_p=dev(p, torch.float32), min_p=dev(least, torch.float32), **kw)
    return tok.cpu().numpy(), lp.cpu().numpy()


def _check(x, u, t=None, k=None, p=None, least=None):
    tok, lp = _run(x, u, t, k, p, least)
    h = x.float().cpu().numpy()
    f = lambda v, off: off if v is None else v  # noqa: E731
    for r in range(len(u)):
        one = [np.float32(f(v, [off] * len(u))[r]) for v, off in ((t, 1.0), (p, 1.0), (least, 0.0))]
        want = _want(h[r], float(np.float32(u[r])), float(one[0]), f(k, [0] * len(u))[r], float(one[1]), float(one[2]))
        assert tok[r] == want[0], (r, tok[r], want, [f(v, [None] * len(u))[r] for v in (t, k, p, least)])
        # one rounding of the logarithm, and weights held to 2^-45 of the largest
        if math.isfinite(want[1]):
            assert abs(lp[r] - want[1]) <= 2.0 ** -24 * abs(want[1]) + 2.0 ** -44 * (1 + math.exp(-max(want[1], -30))), (r, lp[r], want)
        else:
            assert lp[r] == want[1]


def _rows(rows, vocab, sigma=2.5, peaked=True, dtype=None, seed=0):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = sigma * torch.randn(rows, vocab, generator=g, device="cuda")
    if peaked:
        n = min(30, vocab)
        x.scatter_add_(1, torch.randint(0, vocab, (rows, n), generator=g, device="cuda"),
                       4 + 8 * torch.rand(rows, n, generator=g, device="cuda"))
    return x.to(dtype) if dtype else x


@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 1000, 2049, 4096, 16385, 32000, 50257, 201088, 400000])
def test_vocabularies_and_settings(vocab):
    rng = np.random.default_rng(vocab)
    n = 24
    x = _rows(n, vocab, seed=vocab)
    _check(x, rng.random(n), t=rng.choice([0.0, 0.3, 0.7, 1.0, 2.0], n), k=rng.choice([0, 1, 5, 50, 3000, vocab], n),
           p=rng.choice([1.0, 0.0, 0.3, 0.9, 0.99], n), least=rng.choice([0.0, 0.01, 0.2, 1.0, 1.5], n))


@pytest.mark.parametrize("kind", ["none", "temperature", "top_k", "top_p", "min_p"])
@pytest.mark.parametrize("peaked", [True, False])
def test_each_filter_alone(kind, peaked):
    rng = np.random.default_rng(5)
    n = 16
    x = _rows(n, 40000, sigma=1.0, peaked=peaked, seed=6)
    u = rng.random(n)
    if kind == "none":
        _check(x, u)
    elif kind == "temperature":
        _check(x, u, t=rng.uniform(0.1, 5.0, n))
    elif kind == "top_k":
        _check(x, u, k=rng.integers(2, 39999, n))
    elif kind == "top_p":
        _check(x, u, p=rng.uniform(0.01, 0.9999, n))
    else:
        _check(x, u, least=rng.uniform(0.001, 1.0, n))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_16_bit_logits_with_their_ties(dtype):
    """16-bit rows have many equal logits: a cut inside a tie goes by id."""
    import torch

    rng = np.random.default_rng(7)
    n = 32
    x = _rows(n, 30000, sigma=0.5, peaked=False, dtype=getattr(torch, dtype), seed=8)
    _check(x, rng.random(n), k=rng.integers(2, 20000, n))
    _check(x, rng.random(n), p=rng.uniform(0.05, 0.95, n))
    _check(x, rng.random(n), k=rng.integers(2, 5000, n), p=rng.uniform(0.05, 0.95, n), t=rng.uniform(0.3, 2, n))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [1500, 150001])
@pytest.mark.parametrize("offset", [0.0, 250.0, -1000.0])
def test_top_p_over_many_tokens(vocab, dtype, offset):
    """Cuts among thousands of tokens, flat and peaked rows, quantised ones (a
    tie of many at the cut), offsets that cost the histograms' grid its
    precision, behind a large top-k and before a min-p."""
    import torch

    rng = np.random.default_rng(vocab)
    n = 32
    x = torch.cat([_rows(n // 4, vocab, sigma=s, peaked=pk, seed=77 + i)
                   for i, (s, pk) in enumerate(((0.5, False), (2.0, True), (4.0, False), (1.0, True)))])
    x[::5] = (x[::5] * 4).round() / 4
    x = (x + offset).to(getattr(torch, dtype))
    _check(x, rng.random(n), t=rng.choice([0.05, 0.5, 1.0, 2.0, 20.0], n),
           k=rng.choice([0, 0, 0, 1400, vocab * 3 // 4], n), p=rng.choice([0.05, 0.5, 0.9, 0.99, 0.9999], n),
           least=rng.choice([0.0, 0.0, 1e-4, 0.5], n))


def test_an_infinite_temperature_weighs_what_is_not_masked_equally():
    import torch

    x = torch.full((3, 5000), -math.inf, device="cuda")
    ids = torch.arange(0, 4500, 15, device="cuda")  # 300 tokens
    x[:, ids] = 0.0
    x[1:, ids] = -torch.arange(300, device="cuda", dtype=torch.float32)
    for k in (None, [250] * 3):
        tok, lp = _run(x, [0.999, 0.999, 0.0], t=[math.inf] * 3, k=k, p=[0.2, 0.2, 0.2])
        # 0.2 as f32 is above a fifth (13421773 2^-26): 300 (250) of them leave the weight of
        # 60 (50) tokens below top_p of all, so one more is kept
        kept = 61 if k is None else 51
        assert list(tok) == [15 * (kept - 1), 15 * (kept - 1), 0]
        assert np.allclose(lp, -math.log(kept), rtol=2.0 ** -23)


def test_equal_logits_are_drawn_by_id():
    import torch

    vocab = 20000
    for value in (0.0, -3.5, float("inf"), -1e38):
        x = torch.full((6, vocab), value, device="cuda")
        u = [0.0, 0.25, 0.5, 0.75, 0.99, 1 - 2.0 ** -24]
        tok, lp = _run(x, u)
        assert tok.tolist() == [min(int(v * vocab), vocab - 1) for v in u]
        tok, _ = _run(x, u, k=[1, 10, 1000, 7, 15000, 19999])
        assert tok.tolist() == [0, 2, 500, 5, 14850, 19998]
        tok, _ = _run(x, u, p=[0.5] * 6)
        assert tok.tolist() == [min(int(v * vocab / 2), vocab // 2 - 1) for v in u]


def test_exact_borders():
    """Weights that are powers of two: u on a border takes the token after it."""
    import torch

    ln2 = math.log(2.0)
    x = torch.zeros(4, 4, device="cuda")
    tok, lp = _run(x, [0.0, 0.25, 0.5, 0.75])
    assert tok.tolist() == [0, 1, 2, 3]
    assert np.allclose(lp, -2 * ln2, rtol=2.0 ** -24, atol=0)
    tok, _ = _run(x, [0.9] * 4, p=[0.25, 0.2500001, 0.5, 0.75])  # mass before a token < top_p
    assert tok.tolist() == [0, 1, 1, 2]


def test_masked_rows():
    """-inf, the type's lowest value, NaN and +inf among the logits; rows with
    nothing left."""
    import torch

    rng = np.random.default_rng(9)
    x = _rows(12, 30000, seed=10)
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2] = -float("inf")
    x[2, 12345] = -4.0
    x[3, 100:] = -float("inf")
    x[4, 100:] = torch.finfo(torch.float32).min
    x[5] = torch.finfo(torch.float32).min
    x[6, 7] = float("nan")
    x[7, [5, 20000]] = float("inf")
    x[8, ::2] = -float("inf")
    x[9, 1:] = -float("inf")
    x[10] = -x[10].abs() * 1e30
    x[11] = 0.0
    x[11, ::3] = -0.0
    for kw in (dict(), dict(k=[50] * 12), dict(p=[0.9] * 12), dict(least=[0.05] * 12), dict(t=[0.0] * 12),
               dict(k=[150] * 12, p=[0.8] * 12, least=[0.01] * 12, t=[0.7] * 12), dict(t=[1e-30] * 12, p=[0.5] * 12),
               dict(t=[1e30] * 12, k=[20000] * 12)):
        _check(x, rng.random(12), **kw)


def test_uniform_numbers_outside_their_range():
    x = _rows(6, 5000, seed=11)
    x[:] = x[:1]
    tok, _ = _run(x, [-1.0, float("nan"), 0.0, 1.0, 2.0, 1 - 2.0 ** -24])
    assert tok[0] == tok[1] == tok[2] and tok[3] == tok[4]
    assert tok[3] >= tok[5]


def test_strided_and_unaligned_rows_and_many_rows():
    import torch

    rng = np.random.default_rng(12)
    wide = _rows(300, 3001, seed=13)
    for x in (wide[:, 1:3000], wide[:, :2999], wide.bfloat16()[:, 3:2003], wide[::2, 4:1004]):
        n = x.shape[0]
        _check(x, rng.random(n), k=rng.integers(0, 100, n), p=rng.uniform(0.5, 1.0, n))
    out = torch.full((300,), -7, dtype=torch.int32, device="cuda")
    lp = torch.empty(300, device="cuda")
    tok, _ = sampling.sample(wide, torch.rand(300, device="cuda"), tokens=out, logprobs=lp)
    assert tok is out and (out >= 0).all()
    e, _ = sampling.sample(wide[:0], torch.rand(0, device="cuda"))
    assert e.numel() == 0


def test_draws_follow_the_distribution():
    """A grid of u over one row gives each kept token its share to 1 / n."""
    import torch

    n = 4096
    x = _rows(1, 300, sigma=1.0, peaked=False, seed=14).expand(n, 300).contiguous()
    u = (torch.arange(n) + 0.5) / n
    tok, lp = _run(x, u, p=[0.8] * n)
    got = np.bincount(tok, minlength=300) / n
    share = np.zeros(300)
    share[tok] = np.exp(lp)
    assert np.abs(got - share).max() <= 1.0 / n + 1e-6 and abs(share.sum() - 1) < 1e-4


def test_graph_replay_and_another_stream():
    import torch

    x, u = _rows(5, 50000, seed=15), torch.rand(5, device="cuda")
    k = torch.tensor([0, 40, 40, 0, 7], dtype=torch.int32).cuda()
    p = torch.tensor([0.9, 1.0, 0.8, 1.0, 0.5]).cuda()
    tok, lp = torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty(5, device="cuda")
    go = lambda: sampling.sample(x, u, top_k=k, top_p=p, tokens=tok, logprobs=lp)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(10):
        x.normal_(0, 3)
        u.uniform_()
        graph.replay()
        a, b = tok.clone(), lp.clone()
        go()
        assert torch.equal(a, tok) and torch.equal(b, lp)


def test_python_refusals():
    import torch

    x, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    for call in (lambda: sampling.sample(x, u[:1]), lambda: sampling.sample(x, u.double()),
                 lambda: sampling.sample(x.T, u), lambda: sampling.sample(x, u, top_k=u),
                 lambda: sampling.sample(x.double(), u), lambda: sampling.sample(x, u.cpu()),
                 lambda: sampling.sample(x, u, temperature=torch.ones(4, device="cuda")[::2])):
        with pytest.raises(GalliumError):
            call()
