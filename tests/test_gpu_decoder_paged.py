"""gb_decoder_forward_paged: the GPT-OSS decode stack over a paged cache and a
ragged batch, against one numpy oracle (oracle/decoder_oracle.py) per sequence.
Prompts, chunks of prompts and single tokens in one call, sequences without
tokens, a fork that shares pages, sampled continuations, a captured step, and
the refusals."""
import math

import numpy as np
import pytest

from gallium_b200 import GalliumError, GptOssQ, _lib, paged, sampling, synth
from oracle import decoder_oracle as dor

pytestmark = pytest.mark.gpu

PAGE, MAX_SEQ = 8, 96


def _weights(seed, head_dim=64, layers=2):
    # every expert is active, so a rounding cannot change which experts a row takes
    return synth.gptoss_decoder(n_layers=layers, hidden=256, n_heads=8, n_kv_heads=2, head_dim=head_dim,
                                vocab=1000, n_experts=4, top_k=4, inter=256, sliding_window=8, seed=seed)


class Oracle(dor.OracleDecoder):
    """One sequence; queries, keys and values rounded to the pools' type
    (round: None keeps them in f32), and the weights of a softmax as well."""

    def __init__(self, weights, dtype):
        super().__init__(weights, MAX_SEQ)
        self.dtype = dtype

    def copy(self):
        o = object.__new__(Oracle)
        o.__dict__.update(self.__dict__)
        o.k, o.v = list(self.k), list(self.v)
        return o

    def _round(self, x):
        import torch

        x = np.ascontiguousarray(x, np.float32)
        return x if self.dtype is None else torch.from_numpy(x).to(self.dtype).float().numpy()

    def _attention(self, l, x, pos):
        w, L, P = self.w, self.w.layers[l], self.lw[l]
        T, nh, nkv, hd = x.shape[1], w.n_heads, w.n_kv_heads, w.head_dim
        q, k, v = (self._linear(x[0], P[n], b).reshape(T, -1, hd).transpose(1, 0, 2)
                   for n, b in (("wq", L.bq), ("wk", L.bk), ("wv", L.bv)))
        cos, sin = self.cos[pos:pos + T], self.sin[pos:pos + T]
        q, k, v = self._round(dor.rope(q, cos, sin)), self._round(dor.rope(k, cos, sin)), self._round(v)
        K = self.k[l] = k if self.k[l] is None else np.concatenate([self.k[l], k], axis=1)
        V = self.v[l] = v if self.v[l] is None else np.concatenate([self.v[l], v], axis=1)
        out = np.empty((T, nh, hd))
        for h in range(nh):
            s = q[h].astype(np.float64) @ K[h * nkv // nh].astype(np.float64).T / math.sqrt(hd)
            for t in range(T):
                ok = dor.visible(pos + t, K.shape[1], bool(L.sliding), w.sliding_window)
                row = np.where(ok, s[t], -np.inf)
                m = max(row.max(), float(L.sinks[h]))
                e = np.exp(row - m)
                total = e.sum() + math.exp(float(L.sinks[h]) - m)
                out[t, h] = self._round(e).astype(np.float64) @ V[h * nkv // nh] / total
        return self._linear(out.reshape(1, T, -1).astype(np.float32), P["wo"], L.bo)


class Serve:
    """Sequences over one PagePool, each with an oracle in the pools' type and one in f32."""

    def __init__(self, model, w, dtype, n_pages=64):
        import torch

        self.m, self.w = model, w
        self.pool = paged.PagePool(n_pages, PAGE)
        shape = (w.n_layers, n_pages, PAGE, w.n_kv_heads, w.head_dim)
        self.k = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        self.v = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        self.dtype, self.oracles = dtype, {}

    def add(self):
        s = self.pool.add()
        self.oracles[s] = (Oracle(self.w, self.dtype), Oracle(self.w, None))
        return s

    def fork(self, s):
        t = self.pool.fork(s)
        self.oracles[t] = tuple(o.copy() for o in self.oracles[s])
        return t

    def batch(self, seqs, lens, pad=0):
        import torch

        copies = ([], [])
        for s, n in zip(seqs, lens):
            src, dst = self.pool.extend(s, n)
            copies[0].extend(src)
            copies[1].extend(dst)
        if copies[0]:
            paged.copy_pages(list(self.k) + list(self.v), *copies)
        table = np.full((len(seqs), MAX_SEQ // PAGE), -1, np.int32)
        for i, s in enumerate(seqs):
            pages = self.pool.pages(s)
            table[i, :len(pages)] = pages
        put = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()
        return paged.PagedBatch(put(np.concatenate([[0], np.cumsum(lens)])),
                                put([self.pool.length(s) for s in seqs]), put(table), page_size=PAGE,
                                total_q=sum(lens) + pad, max_q_len=max(lens), max_kv_len=MAX_SEQ)

    def step(self, seqs, tokens, pad=0):
        """tokens: one array per sequence.  Checks the logits, returns them."""
        lens = [len(t) for t in tokens]
        b = self.batch(seqs, lens, pad)
        ids = np.concatenate([np.asarray(t, np.int32) for t in tokens] + [np.zeros(pad, np.int32)])
        logits = self.m.forward_paged(ids, b, self.k, self.v)
        got = logits.cpu().numpy()
        assert np.array_equal(self.m.last_next.cpu().numpy(), dor.greedy(got))
        for i, s in enumerate(seqs):
            if not lens[i]:
                assert not got[i].any()
                continue
            near, exact = (o.forward(np.asarray(tokens[i])[None], o.pos)[0] for o in self.oracles[s])
            # What the roundings of q, k, v and the weights to the pools' type move the logits
            # by is `moved`.  The kernels round the same values at the same places, but from
            # f32 sums in another order and with weights taken against another maximum: where
            # that falls on the other side of a rounding the difference is one more rounding
            # of the same kind, so the distance is at most of the size of `moved` again; the
            # stack's own f32 tolerance (2e-2 of the largest error, 1e-3 of the mean) comes on top.
            moved = np.abs(near - exact)
            err = np.abs(got[i].astype(np.float64) - near)
            assert err.max() <= 2 * moved.max() + 2e-2, (s, err.max(), moved.max())
            assert err.mean() <= 2 * moved.mean() + 1e-3 * np.abs(near).mean(), (s, err.mean(), moved.mean())
        return logits


def _load(w, max_batch=4, max_tokens=12):
    return GptOssQ.load(w, device=0, max_batch=max_batch, max_tokens=max_tokens, max_seq_len=MAX_SEQ)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_ragged_prompts_chunks_and_steps(head_dim, dtype):
    import torch

    w = _weights(3, head_dim)
    rng = np.random.default_rng(head_dim)
    tok = lambda n: rng.integers(0, w.vocab, n).astype(np.int32)
    with _load(w) as m:
        sv = Serve(m, w, getattr(torch, dtype))
        a, b, c = sv.add(), sv.add(), sv.add()
        sv.step([a, b, c], [tok(21), tok(1), tok(0)])          # a prompt, one token, nothing yet
        sv.step([c, a], [tok(17), tok(1)])                     # a prompt beside a decoding step
        d = sv.fork(a)
        sv.step([a, d, b, c], [tok(1), tok(1), tok(20), tok(9)], pad=3)
        for _ in range(3):
            sv.step([d, c, b, a], [tok(1)] * 4)
        sv.step([b], [tok(1)])


def test_a_batch_without_new_tokens():
    import torch

    w = _weights(11, layers=1)
    with _load(w) as m:
        sv = Serve(m, w, torch.bfloat16)
        a, b = sv.add(), sv.add()
        for rows in (0, 4):  # rows of no sequence
            torch.full((2, w.vocab), 3.0, device="cuda")  # what an unwritten result would hold
            batch = paged.PagedBatch(torch.zeros(3, dtype=torch.int32, device="cuda"),
                                     torch.zeros(2, dtype=torch.int32, device="cuda"),
                                     torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), page_size=PAGE,
                                     total_q=rows, max_q_len=0, max_kv_len=MAX_SEQ)
            logits = m.forward_paged(np.zeros(rows, np.int32), batch, sv.k, sv.v)
            assert not logits.any() and list(m.last_next.cpu()) == [w.vocab - 1] * 2
        sv.step([a, b], [np.arange(5), np.arange(3)])


def test_own_cache_and_paged_forwards_do_not_disturb_each_other():
    import torch

    w = _weights(5)
    toks = np.random.default_rng(5).integers(0, w.vocab, (2, 6)).astype(np.int32)
    with _load(w) as m:
        x = torch.from_numpy(toks).cuda()
        m.forward(x, 0)
        start = m.last_next.clone()
        want = m.generate(start, 6, 5).cpu().numpy()
        m.reset()
        m.forward(x, 0)
        sv = Serve(m, w, torch.bfloat16)
        s = sv.add()
        sv.step([s], [toks[0]])
        assert np.array_equal(m.generate(start, 6, 5).cpu().numpy(), want)
        sv.step([s], [toks[1, :1]])


def test_sampled_continuation_and_a_captured_step():
    """A decoding step (forward, sampling) captured once and replayed with the
    lengths, tokens and uniforms moved on in place, against eager steps."""
    import torch

    w = _weights(7)
    rng = np.random.default_rng(7)
    steps, n = 6, 3
    u = torch.from_numpy(rng.random((steps, n), dtype=np.float32)).cuda()
    t = torch.tensor([0.7, 0.0, 1.3], device="cuda")
    k = torch.tensor([0, 0, 20], dtype=torch.int32, device="cuda")
    p = torch.tensor([0.9, 1.0, 0.95], device="cuda")
    prompts = [rng.integers(0, w.vocab, c).astype(np.int32) for c in (9, 2, 15)]
    with _load(w) as m:
        outs = []
        for captured in (False, True):
            sv = Serve(m, w, torch.bfloat16)
            seqs = [sv.add() for _ in range(n)]
            logits = sv.step(seqs, prompts)
            first = sampling.sample(logits, u[0], temperature=t, top_k=k, top_p=p)[0]
            batch = sv.batch(seqs, [steps] * n)  # pages for all steps
            batch = paged.PagedBatch(torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                                     batch.kv_len - (steps - 1), batch.page_table, page_size=PAGE,
                                     total_q=n, max_q_len=1, max_kv_len=MAX_SEQ)
            tokens, draw = first.clone(), u[1].clone()

            def step():
                lg = m.forward_paged(tokens, batch, sv.k, sv.v, check_status=False)
                sampling.sample(lg, draw, temperature=t, top_k=k, top_p=p, tokens=tokens)

            if captured:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    step()
            out = [first.cpu().numpy()]
            for i in range(1, steps):
                draw.copy_(u[i])
                g.replay() if captured else step()
                batch.kv_len.add_(1)
                out.append(tokens.cpu().numpy().copy())
            batch.check()
            outs.append(np.stack(out))
        assert np.array_equal(outs[0], outs[1])
        # the row at temperature 0 follows its oracle's greedy tokens
        for i in range(steps - 1):
            near, exact = (o.forward(outs[0][i, 1:2][None], o.pos)[0] for o in sv.oracles[seqs[1]])
            # only a near-tie may go the other way: two logits, each off by Serve.step's bound
            assert near.max() - near[outs[0][i + 1, 1]] <= 2 * (2 * np.abs(near - exact).max() + 2e-2)


def test_refusals_and_flags():
    import torch

    w = _weights(9, layers=1)
    with _load(w, max_batch=2, max_tokens=4) as m:
        sv = Serve(m, w, torch.bfloat16)
        a, b, c = sv.add(), sv.add(), sv.add()

        def refused(call, status=_lib.GB_ERR_INVALID_ARG):
            with pytest.raises(GalliumError) as e:
                call()
            assert e.value.status == status

        ok = sv.batch([a, b], [3, 1])
        ids = np.zeros(4, np.int32)
        refused(lambda: m.forward_paged(ids[:3], ok, sv.k, sv.v))       # tokens of three rows
        refused(lambda: m.forward_paged(ids, ok, sv.k[:0], sv.v))       # no pool for the layer
        refused(lambda: m.forward_paged(ids, ok, sv.k[..., :32], sv.v[..., :32]),
                _lib.GB_ERR_UNSUPPORTED)                                # head_dim 32
        wide = torch.zeros((1, 64, PAGE, 2, 128), dtype=torch.bfloat16, device="cuda")
        refused(lambda: m.forward_paged(ids, ok, wide, wide.clone()))   # not the model's head_dim
        three = sv.batch([a, b, c], [1, 1, 1])
        refused(lambda: m.forward_paged(ids[:3], three, sv.k, sv.v))    # more sequences than max_batch
        long = sv.batch([a, b], [8, 1])
        refused(lambda: m.forward_paged(np.zeros(9, np.int32), long, sv.k, sv.v))  # more rows than fit
        m.forward_paged(ids, ok, sv.k, sv.v)
        refused(lambda: m.forward_paged(np.full(4, w.vocab, np.int32), ok, sv.k, sv.v))  # token ids
        m.forward_paged(ids, ok, sv.k, sv.v)
        ok.page_table[0, 0] = 64  # outside the pool
        refused(lambda: m.forward_paged(ids, ok, sv.k, sv.v))
        ok.page_table[0, 0] = sv.pool.pages(a)[0]
        ok.kv_len.add_(MAX_SEQ)  # past max_seq_len and the batch's bound
        refused(lambda: m.forward_paged(ids, ok, sv.k, sv.v))
