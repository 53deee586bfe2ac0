"""The serving operators around a paged KV cache, case by case: what each
computes in plain torch operations, what it has to move, and the call that a
program makes of this package.

  rope_append   RMS norm of each query and key head, position rotation, keys and
                values stored into the pages of their sequence, in one pass
  attention     a ragged batch of new tokens (chunks, single tokens, or both)
                over each sequence's pages: causal, grouped queries, an optional
                sliding window, an optional sink logit per query head
  copy_pages    pages of every layer's pools copied to other pages (a fork's
                last page, a compaction)
  sample        one token per row of logits from a given uniform number, under
                temperature, top-k, top-p and min-p

Sequence b has rows q_start[b] .. q_start[b + 1] of the batch and kv_len[b]
cached positions, its own new ones included: row i of it sits at position
kv_len[b] - q_len[b] + i.  Position p is slot p % page of page
page_table[b][p // page].
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one stream, one token on a sliding layer of the GPT-OSS stack (64 query
        # heads, 8 KV heads of 64): latency alone
        dict(name="rope decode 1", op="rope_append", dtype="bf16", heads=64, kv_heads=8, dim=64, rot=64,
             norm=False, page=16, seqs=1, q_lo=1, q_hi=1, ctx_lo=1000, ctx_hi=1000, decode=1.0, lens=1),
        # a step of 61 streams with query and key norms, f16
        dict(name="rope decode 61", op="rope_append", dtype="f16", heads=32, kv_heads=8, dim=128, rot=128,
             norm=True, page=32, seqs=61, q_lo=1, q_hi=1, ctx_lo=1, ctx_hi=500, decode=1.0, lens=2),
        # prefill of four prompts with query and key norms
        dict(name="rope prefill 8k", op="rope_append", dtype="bf16", heads=32, kv_heads=8, dim=128, rot=128,
             norm=True, page=64, seqs=4, q_lo=2000, q_hi=2048, ctx_lo=0, ctx_hi=64, decode=0.0, lens=3),
        # one stream, one token, a full layer of the GPT-OSS stack at 4 K positions
        dict(name="attn decode 1", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=64, window=0,
             sinks=True, page=16, seqs=1, q_lo=1, q_hi=1, ctx_lo=4096, ctx_hi=4096, decode=1.0, lens=4),
        # a step of 64 streams whose lengths differ by a factor of 16
        dict(name="attn decode 64", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=64, window=0,
             sinks=True, page=64, seqs=64, q_lo=1, q_hi=1, ctx_lo=512, ctx_hi=8192, decode=1.0, lens=5),
        # 24 decoding streams with the chunks of 6 prompts in the same batch, a sliding layer
        dict(name="attn mixed window", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=64, window=128,
             sinks=True, page=16, seqs=30, q_lo=100, q_hi=700, ctx_lo=0, ctx_hi=2000, decode=0.8, lens=6),
        # a prompt's chunk of about a thousand tokens behind 16 K cached ones, f16, heads of 128
        dict(name="attn chunk 16k", op="attention", dtype="f16", heads=32, kv_heads=8, dim=128, window=0,
             sinks=False, page=32, seqs=1, q_lo=1000, q_hi=1024, ctx_lo=16000, ctx_hi=16384, decode=0.0, lens=7),
        # prefill of four prompts, a full layer of the GPT-OSS stack
        dict(name="attn prefill 8k", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=64, window=0,
             sinks=True, page=64, seqs=4, q_lo=1900, q_hi=2048, ctx_lo=0, ctx_hi=0, decode=0.0, lens=8),
        # three forks of a stream: their half-filled last page in 24 layers' K and V
        dict(name="copy fork", op="copy_pages", dtype="bf16", kv_heads=8, dim=64, page=16, pools=48,
             pages=64, moved=3, lens=9),
        # a compaction that moves 301 pages of every layer
        dict(name="copy compact", op="copy_pages", dtype="bf16", kv_heads=8, dim=64, page=64, pools=48,
             pages=700, moved=301, lens=10),
        # one stream, every filter on
        dict(name="sample 1", op="sample", dtype="f32", rows=1, vocab=201088, sigma=2.5, peaked=True,
             settings="all", lens=11),
        # 128 streams, each with its own settings
        dict(name="sample 128", op="sample", dtype="f32", rows=128, vocab=201088, sigma=2.5, peaked=True,
             settings="mixed", lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope_append", "attention", "attention", "copy_pages", "sample", "sample"))
    case = dict(op=op, lens=rng.randrange(1 << 30))
    if op == "sample":
        case.update(dtype=rng.choice(("f32", "f32", "bf16", "f16")), rows=_log(rng, 1, 128),
                    vocab=_log(rng, 1000, 262144), sigma=round(rng.uniform(0.5, 4.0), 2),
                    peaked=rng.random() < 0.7, settings=rng.choice(("all", "mixed", "none")))
        case["rows"] = max(1, min(case["rows"], 25_000_000 // case["vocab"]))
        return case
    case.update(dtype=rng.choice(("bf16", "f16")), dim=rng.choice((64, 64, 128, 256)),
                page=rng.choice((16, 32, 64, 128)), kv_heads=rng.choice((1, 2, 4, 8)))
    if op == "copy_pages":
        case.update(pools=_log(rng, 2, 96), moved=_log(rng, 1, 300))
        page_bytes = 2 * case["page"] * case["kv_heads"] * case["dim"]
        case["moved"] = max(1, min(case["moved"], 900_000_000 // (page_bytes * case["pools"])))
        case["pages"] = 2 * case["moved"] + rng.randrange(1, 40)
        return case
    case["heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4, 5, 7, 8))
    if op == "rope_append":
        case.update(rot=rng.choice((case["dim"], case["dim"], case["dim"] // 2)), norm=rng.random() < 0.6)
    else:
        case.update(window=rng.choice((0, 0, 0, 100, 128, 1000)), sinks=rng.random() < 0.5)
    kind = rng.choice(("decode", "chunk", "mixed"))
    if kind == "decode":
        case.update(seqs=_log(rng, 1, 128), q_lo=1, q_hi=1, ctx_lo=0, ctx_hi=_log(rng, 100, 16000), decode=1.0)
    elif kind == "chunk":
        case.update(seqs=_log(rng, 1, 8), q_lo=0, q_hi=_log(rng, 2, 2048), ctx_lo=0, ctx_hi=_log(rng, 1, 8000),
                    decode=0.0)
    else:
        case.update(seqs=_log(rng, 8, 64), q_lo=2, q_hi=_log(rng, 8, 500), ctx_lo=0, ctx_hi=_log(rng, 10, 3000),
                    decode=0.7)
    # the plain form's padded scores, and the pools, stay under a few GB
    while (case["seqs"] * case["heads"] * case["q_hi"] * (case["q_hi"] + case["ctx_hi"]) > 1 << 29
           or case["seqs"] * case["kv_heads"] * case["dim"] * (case["q_hi"] + case["ctx_hi"]) > 1 << 28):
        if case["seqs"] > 1 and case["seqs"] >= case["q_hi"] // 64:
            case["seqs"] = (case["seqs"] + 1) // 2
        else:
            case["ctx_hi"] = (case["ctx_hi"] + 1) // 2
            if case["decode"] < 1.0:
                case["q_hi"] = (case["q_hi"] + 1) // 2
    case["q_lo"] = min(case["q_lo"], case["q_hi"])
    return case


def _lengths(case):
    """[(new tokens, cached positions with them)] of each sequence."""
    r = random.Random(case["lens"])
    got = []
    for b in range(case["seqs"]):
        q = 1 if r.random() < case["decode"] else r.randint(case["q_lo"], case["q_hi"])
        lo, hi = case["ctx_lo"], case["ctx_hi"]
        ctx = lo if hi <= lo else int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1
        got.append((q, q + ctx))
    if not sum(q for q, _ in got):
        got[0] = (1, got[0][1] + 1)
    return got


def _paged(case, g, dev):
    """The batch: sequences' lengths and pages, in an order that a long-running cache has."""
    lens = _lengths(case)
    need = [-(-kv // case["page"]) for _, kv in lens]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    width = max(max(need), 1)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    n = torch.tensor(need, device=dev)
    at = torch.cumsum(n, 0) - n
    col = torch.arange(width, device=dev)
    table = torch.where(col < n[:, None], order[(at[:, None] + col).clamp(max=n_pages - 1)], table)
    q = torch.tensor([0] + [x for x, _ in lens], dtype=torch.int32)
    s = dict(lens=lens, n_pages=n_pages, table=table.contiguous(), page=case["page"],
             q_start=torch.cumsum(q, 0).to(torch.int32).to(dev),
             kv_len=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=dev),
             total_q=sum(x for x, _ in lens), max_q=max(x for x, _ in lens),
             max_kv=max(kv for _, kv in lens))
    if own:
        s["batch"] = _api("paged").PagedBatch(s["q_start"], s["kv_len"], s["table"], page_size=s["page"],
                                              total_q=s["total_q"], max_q_len=s["max_q"],
                                              max_kv_len=s["max_kv"])
    return s


def _api(name):
    import importlib

    path = os.path.join(os.getcwd(), "rs-gallium_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    return importlib.import_module("gallium_b200." + name)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def normal(*shape, dtype=t, std=1.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, std, generator=g)

    if case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        x = torch.randn(R, V, generator=g, device=dev) * case["sigma"]
        if case["peaked"]:  # a trained model's rows: a few dozen tokens far above the rest
            n = min(40, V)
            at = torch.randint(0, V, (R, n), generator=g, device=dev)
            x.scatter_add_(1, at, 4 + 10 * torch.rand(R, n, generator=g, device=dev))
        s = dict(op="sample", x=x.to(t), u=torch.rand(R, generator=g, device=dev), temperature=None,
                 top_k=None, top_p=None, min_p=None)
        if case["settings"] == "all":
            s.update(temperature=torch.full((R,), 0.8, device=dev),
                     top_k=torch.full((R,), 50, dtype=torch.int32, device=dev),
                     top_p=torch.full((R,), 0.9, device=dev), min_p=torch.full((R,), 0.02, device=dev))
        elif case["settings"] == "mixed":
            def pick(values, dtype):
                return torch.tensor(values, dtype=dtype, device=dev)[
                    torch.randint(0, len(values), (R,), generator=g, device=dev)]
            s.update(temperature=pick([0.0, 0.6, 0.7, 0.8, 1.0, 1.3], torch.float32),
                     top_k=pick([0, 0, 20, 40, 64, 1000], torch.int32),
                     top_p=pick([1.0, 0.8, 0.9, 0.95, 0.99], torch.float32),
                     min_p=pick([0.0, 0.0, 0.02, 0.1], torch.float32))
        return s
    kvh, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "copy_pages":
        pools = normal(case["pools"], case["pages"], page, kvh, dim)
        order = torch.randperm(case["pages"], generator=g, device=dev).tolist()
        n = case["moved"]
        return dict(op="copy_pages", pools=pools, src=order[:n], dst=order[n:2 * n])
    s = _paged(case, g, dev)
    N, H = s["total_q"], case["heads"]
    s.update(op=case["op"], k_pool=normal(s["n_pages"], page, kvh, dim),
             v_pool=normal(s["n_pages"], page, kvh, dim))
    if case["op"] == "rope_append":
        qkv = normal(N, (H + 2 * kvh) * dim, std=2.0)  # one projection's rows, q heads then k then v
        s.update(q=qkv[:, :H * dim].view(N, H, dim), k=qkv[:, H * dim:(H + kvh) * dim].view(N, kvh, dim),
                 v=qkv[:, (H + kvh) * dim:].view(N, kvh, dim), eps=1e-6, rot=case["rot"], q_norm=None, k_norm=None)
        if case["norm"]:
            s.update(q_norm=1 + normal(dim, dtype=torch.float32, std=0.2),
                     k_norm=1 + normal(dim, dtype=torch.float32, std=0.2))
        freq = 150000.0 ** (-torch.arange(case["rot"] // 2, dtype=torch.float64, device=dev) * 2 / case["rot"])
        angle = torch.arange(s["max_kv"], dtype=torch.float64, device=dev)[:, None] * freq
        s.update(cos=angle.cos().float(), sin=angle.sin().float())
        return s
    s.update(q=normal(N, H, dim), window=case["window"], scale=1.0 / math.sqrt(dim),
             sinks=normal(H, dtype=torch.float32) if case["sinks"] else None)
    return s


def run(s):
    op = s["op"]
    if own:
        if op == "rope_append":
            q = _paged_api().rope_append(s["batch"], s["q"], s["k"], s["v"], s["k_pool"], s["v_pool"], s["cos"],
                                         s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"])
            return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
        if op == "attention":
            return {"out": _paged_api().attention(s["batch"], s["q"], s["k_pool"], s["v_pool"], sinks=s["sinks"],
                                                  window=s["window"], scale=s["scale"])}
        if op == "copy_pages":
            _paged_api().copy_pages(s["pools"], s["src"], s["dst"])
            return {"pools": s["pools"]}
        token, logprob = _sample_api().sample(s["x"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                              top_p=s["top_p"], min_p=s["min_p"])
        return {"token": token, "logprob": logprob}
    if op == "rope_append":
        return _plain_rope_append(s)
    if op == "attention":
        return {"out": _plain_attention(s)}
    if op == "copy_pages":
        src, dst = (torch.tensor(v, device=s["pools"].device) for v in (s["src"], s["dst"]))
        s["pools"][:, dst] = s["pools"][:, src]
        return {"pools": s["pools"]}
    return _plain_sample(s)


_MODULES = {}


def _paged_api():
    if "paged" not in _MODULES:
        _MODULES["paged"] = _api("paged")
    return _MODULES["paged"]


def _sample_api():
    if "sampling" not in _MODULES:
        _MODULES["sampling"] = _api("sampling")
    return _MODULES["sampling"]


def _rows(s):
    """Each row's sequence and position."""
    row = torch.arange(s["total_q"], device=s["q_start"].device, dtype=torch.int32)
    b = torch.searchsorted(s["q_start"][1:].contiguous(), row, right=True)
    return b, (row - s["q_start"][b + 1] + s["kv_len"][b]).long()


def _plain_rope_append(s):
    b, pos = _rows(s)
    half = s["rot"] // 2
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * w
        x1, x2 = x[..., :half], x[..., half:2 * half]
        return torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos, x[..., 2 * half:]], -1).to(s["q"].dtype)

    page, slot = s["table"][b, pos // s["page"]].long(), pos % s["page"]
    s["k_pool"][page, slot] = turned(s["k"], s["k_norm"])
    s["v_pool"][page, slot] = s["v"]
    return {"q": turned(s["q"], s["q_norm"]), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_attention(s):
    q = s["q"]
    N, H, dim = q.shape
    B, kvh = s["kv_len"].numel(), s["k_pool"].shape[2]
    dev = q.device
    pages = s["table"].clamp(min=0).long()
    keys, values = (s[p][pages].flatten(1, 2)[:, :s["max_kv"]].float().transpose(1, 2) for p in ("k_pool", "v_pool"))
    b, pos = _rows(s)
    row = torch.arange(N, device=dev) - s["q_start"][b]
    padded = torch.zeros(B, s["max_q"], H, dim, device=dev)
    padded[b, row] = q.float()
    at = torch.full((B, s["max_q"]), -1, dtype=torch.long, device=dev)
    at[b, row] = pos
    # scores of [sequence, KV head, query head of its group and row, key]
    padded = padded.view(B, s["max_q"], kvh, H // kvh, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = (padded @ keys.transpose(2, 3)).mul_(s["scale"]).view(B, kvh, H // kvh, s["max_q"], -1)
    key = torch.arange(keys.shape[2], device=dev)
    seen = key <= at[..., None]
    if s["window"]:
        seen &= key > at[..., None] - s["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, kvh, H // kvh, 1, 1)
        top = torch.maximum(top, sink)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - top).exp()
    out = (p.flatten(2, 3) @ values).view(B, kvh, H // kvh, s["max_q"], dim) / total.masked_fill(total == 0, 1.0)
    return out.permute(0, 3, 1, 2, 4).reshape(B, s["max_q"], H, dim)[b, row].to(q.dtype)


def _plain_sample(s):
    x, u = s["x"].double(), s["u"].double()
    R, V = x.shape
    dev = x.device

    def given(name, off):
        v = s[name]
        return torch.full((R, 1), off, dtype=torch.float64, device=dev) if v is None else v.double()[:, None]

    t, k, p, least = given("temperature", 1.0), given("top_k", 0), given("top_p", 1.0), given("min_p", 0.0)
    greedy = t <= 0
    value, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lowest id first
    rank = torch.arange(V, device=dev)[None]
    w = ((value - value[:, :1]) / torch.where(greedy, 1.0, t)).exp()
    w = w * ((k <= 0) | (rank < k))
    before = torch.cumsum(w, 1)
    before = torch.cat([torch.zeros_like(before[:, :1]), before[:, :-1]], 1)
    keep = (p >= 1) | (before < p * w.sum(1, keepdim=True))
    keep &= (w >= least) & (~greedy | (rank < 1))
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, w * keep)  # by token id
    c = torch.cumsum(w, 1)
    token = (c <= u[:, None] * c[:, -1:]).sum(1, keepdim=True).clamp(max=V - 1)
    logprob = (w.gather(1, token) / c[:, -1:]).log()
    return {"token": token[:, 0].to(torch.int32), "logprob": logprob[:, 0].float()}


def exact(case, seed):
    """The same from the definitions in 64 bits, sequence by sequence and row by row."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "copy_pages":
        pools = s["pools"].double()
        for a, b in zip(s["src"], s["dst"]):
            pools[:, b] = s["pools"][:, a].double()
        return {"pools": pools}
    if op == "sample":
        return {"token": None, "logprob": _exact_logprob(s)}
    starts, table = s["q_start"].tolist(), s["table"].tolist()
    if op == "rope_append":
        q, kp, vp = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device), s["k_pool"].double(), s["v_pool"].double()
        z = case["rot"] // 2

        def one(x, w, pos):
            x = x.double()
            if w is not None:
                x = x * w.double() * (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + s["eps"]).rsqrt()
            turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            y = torch.complex(x[..., :z], x[..., z:2 * z]) * turn
            return torch.cat([y.real, y.imag, x[..., 2 * z:]], -1)

        for b, (n, kv) in enumerate(s["lens"]):
            rows = slice(starts[b], starts[b] + n)
            pos = torch.arange(kv - n, kv, device=q.device)
            q[rows] = one(s["q"][rows], s["q_norm"], pos)
            pages = torch.tensor(table[b], device=q.device)[pos // case["page"]].long()
            kp[pages, pos % case["page"]] = one(s["k"][rows], s["k_norm"], pos)
            vp[pages, pos % case["page"]] = s["v"][rows].double()
        return {"q": q, "k_pool": kp, "v_pool": vp}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    group = case["heads"] // case["kv_heads"]
    for b, (n, kv) in enumerate(s["lens"]):
        if not n:
            continue
        pages = torch.tensor(table[b][:-(-kv // case["page"])], device=out.device).long()
        pos = torch.arange(kv - n, kv, device=out.device)[:, None]
        key = torch.arange(kv, device=out.device)[None]
        hidden = (key > pos) | ((pos - key >= case["window"]) if case["window"] else False)
        for h in range(case["heads"]):
            kk, vv = (s[x][pages, :, h // group].double().flatten(0, 1)[:kv] for x in ("k_pool", "v_pool"))
            a = s["q"][starts[b]:starts[b] + n, h].double() @ kk.T * s["scale"]
            a = a.masked_fill(hidden, -math.inf)
            if s["sinks"] is not None:
                a = torch.cat([a, s["sinks"][h].double().expand(n, 1)], 1)
            out[starts[b]:starts[b] + n, h] = torch.softmax(a, 1)[:, :kv] @ vv
    return {"out": out}


def _exact_logprob(s):
    """log of the chosen token's share, row by row on the host; the choice is the definition's too."""
    got = []
    for r in range(s["x"].shape[0]):
        x = s["x"][r].double().cpu()
        at = lambda name, off: off if s[name] is None else float(s[name][r])  # noqa: E731,B023
        t, k, p, least = at("temperature", 1.0), int(at("top_k", 0)), at("top_p", 1.0), at("min_p", 0.0)
        if t <= 0:
            got.append(0.0)
            continue
        order = torch.argsort(x, descending=True, stable=True)
        if k > 0:
            order = order[:k]
        q = torch.softmax(x[order] / t, 0)
        kept = torch.ones(len(order), dtype=torch.bool)
        if p < 1:
            kept[1:] &= torch.cumsum(q, 0)[:-1] < p
        kept[1:] &= q[1:] >= least * q[0]
        order, by_id = torch.sort(order[kept])
        q = q[kept][by_id]
        c = torch.cumsum(q, 0)
        i = int(torch.searchsorted(c, c[-1:] * float(s["u"][r]), right=True).clamp(max=len(c) - 1))
        got.append(math.log(float(q[i] / c[-1])))
    return torch.tensor(got, dtype=torch.float64)


def work(case):
    op, size = case["op"], SIZES[case["dtype"]]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 28, "flops": 4 * n}
    kvh, dim = case["kv_heads"], case["dim"]
    if op == "copy_pages":
        return {"bytes": 2 * size * case["pools"] * case["moved"] * case["page"] * kvh * dim, "flops": 0}
    lens = _lengths(case)
    N, H = sum(q for q, _ in lens), case["heads"]
    if op == "rope_append":
        positions = len({p for q, kv in lens for p in range(kv - q, kv)})
        return {"bytes": 2 * size * N * (H + 2 * kvh) * dim + 4 * case["rot"] * positions + 8 * len(lens),
                "flops": N * (H + kvh) * (3 * case["rot"] + (4 * dim if case["norm"] else 0))}
    window = case["window"] or 1 << 40
    keys = sum(min(kv, window + q - 1) for q, kv in lens if q)
    pairs = 0
    for q, kv in lens:  # visible keys over the sequence's rows: min(position + 1, window)
        first, last = kv - q + 1, kv
        short = max(0, min(last, window) - first + 1)
        pairs += (first + first + short - 1) * short // 2 + (q - short) * min(window, last)
    return {"bytes": 2 * size * (N * H * dim + keys * kvh * dim) + 4 * sum(-(-kv // case["page"]) for _, kv in lens),
            "flops": 4 * dim * H * pairs}
