"""The paged-cache operators and gb_sample without a GPU: struct layouts, the
refusals that come before any device call, the Python checks, and the page
allocator against a plain model of its sequences."""
import ctypes
import random
import subprocess

import numpy as np
import pytest

from gallium_b200 import GalliumError, _lib, paged
from gallium_b200._lib import AttnArgs, PagedBatchDesc, RopeArgs, SampleArgs

BUF = np.zeros(1 << 16, np.uint8)
P = (BUF.ctypes.data + 255) // 256 * 256


def test_struct_layouts_match_the_header(tmp_path):
    src = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{_lib.HEADER_PATH}"', 'int main(void){']
    want = []
    for name, cls in (("gb_paged_batch", PagedBatchDesc), ("gb_rope_args", RopeArgs), ("gb_attn_args", AttnArgs),
                      ("gb_sample_args", SampleArgs)):
        src.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            src.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    src.append("return 0;}")
    c = tmp_path / "layout.c"
    c.write_text("\n".join(src))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", str(c), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


def _set(s, kw):
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _batch(**kw):
    d = PagedBatchDesc()
    return _set(d, dict(dict(struct_size=ctypes.sizeof(d), dtype=_lib.GB_DTYPE_BF16, n_kv_heads=2, head_dim=64,
                             page_size=16, n_pages=4, page_stride=2048, slot_stride=128, head_stride=64, n_seqs=1,
                             total_q=1, max_q_len=1, max_kv_len=8, q_start_dev=P, kv_len_dev=P, page_table_dev=P,
                             table_stride=1), **kw))


def _rope(**kw):
    a = RopeArgs()
    return _set(a, dict(dict(struct_size=ctypes.sizeof(a), in_dtype=_lib.GB_DTYPE_BF16, n_heads=4, rot_dim=64,
                             q_dev=P, k_dev=P, v_dev=P, q_row_stride=512, q_head_stride=64, k_row_stride=512,
                             k_head_stride=64, v_row_stride=512, v_head_stride=64, q_out_dev=P + 4096,
                             out_row_stride=256, out_head_stride=64, cos_dev=P, sin_dev=P, table_rows=8, k_pool_dev=P,
                             v_pool_dev=P, eps=1e-6), **kw))


def _attn(**kw):
    a = AttnArgs()
    return _set(a, dict(dict(struct_size=ctypes.sizeof(a), n_heads=4, window=0, out_dtype=_lib.GB_DTYPE_BF16,
                             scale=0.125, q_dev=P, q_row_stride=256, q_head_stride=64, k_pool_dev=P, v_pool_dev=P,
                             out_dev=P + 4096, out_row_stride=256, out_head_stride=64, workspace_dev=P,
                             workspace_bytes=1 << 40), **kw))


def _sample(**kw):
    a = SampleArgs()
    return _set(a, dict(dict(struct_size=ctypes.sizeof(a), dtype=_lib.GB_DTYPE_F32, rows=2, vocab=100, logits_dev=P,
                             row_stride=100, u_dev=P, token_dev=P), **kw))


def _call(fn, *args):
    lib = _lib.load_library()
    rc = getattr(lib, fn)(*args)
    return rc, lib.gb_last_error().decode()


INV, UNS = _lib.GB_ERR_INVALID_ARG, _lib.GB_ERR_UNSUPPORTED
BATCH_BAD = [
    (dict(struct_size=8), INV, "struct_size"), (dict(dtype=0), UNS, "dtype"), (dict(head_dim=96), UNS, "head_dim"),
    (dict(page_size=24), UNS, "power of two"), (dict(page_size=4), UNS, "power of two"),
    (dict(n_kv_heads=0), INV, "n_kv_heads"), (dict(n_pages=0), INV, "n_pages"), (dict(total_q=-1), INV, ">= 0"),
    (dict(slot_stride=60), INV, "strides"), (dict(head_stride=32), INV, "strides"), (dict(page_stride=4), INV, "strides"),
    (dict(page_stride=-2048), INV, "strides"), (dict(kv_len_dev=None), INV, "kv_len"), (dict(table_stride=-1), INV, "table_stride"),
]


@pytest.mark.parametrize("kw,status,needle", BATCH_BAD)
def test_bad_batches_are_refused_by_both_operators(kw, status, needle):
    b = _batch(**kw)
    for fn, a in (("gb_paged_rope_append", _rope()), ("gb_paged_attention", _attn())):
        rc, msg = _call(fn, ctypes.byref(b), ctypes.byref(a), None)
        assert rc == status and needle in msg, (fn, rc, msg)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(struct_size=1), INV, "struct_size"), (dict(in_dtype=5), INV, "in_dtype"), (dict(n_heads=-1), INV, "n_heads"),
    (dict(rot_dim=24), UNS, "rot_dim"), (dict(rot_dim=80), UNS, "rot_dim"), (dict(eps=-1.0), INV, "eps"),
    (dict(eps=float("nan")), INV, "eps"), (dict(q_dev=None), INV, "null"), (dict(v_pool_dev=None), INV, "null"),
    (dict(cos_dev=None), INV, "cos"), (dict(q_dev=P + 8), INV, "aligned"), (dict(q_norm_dev=P + 4), INV, "aligned"),
    (dict(k_row_stride=130), INV, "strides"), (dict(v_head_stride=-64), INV, "strides"),
    (dict(q_out_dev=P), INV, "q_out"), (dict(table_rows=-1), INV, "table_rows"),
])
def test_rope_append_refuses_bad_arguments(kw, status, needle):
    rc, msg = _call("gb_paged_rope_append", ctypes.byref(_batch()), ctypes.byref(_rope(**kw)), None)
    assert rc == status and needle in msg, (rc, msg)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(struct_size=1), INV, "struct_size"), (dict(n_heads=3), INV, "multiple"), (dict(n_heads=0), INV, "multiple"),
    (dict(n_heads=34), UNS, "at most 16"), (dict(window=-1), INV, "window"), (dict(out_dtype=_lib.GB_DTYPE_F16), UNS, "out_dtype"),
    (dict(scale=0.0), INV, "scale"), (dict(scale=float("inf")), INV, "scale"), (dict(out_dev=None), INV, "null"),
    (dict(out_dev=P), INV, "must not be q"), (dict(q_dev=P + 2), INV, "aligned"), (dict(out_row_stride=4), INV, "strides"),
    (dict(workspace_dev=P + 16), INV, "256-byte"), (dict(workspace_bytes=1000), INV, "needed"),
])
def test_attention_refuses_bad_arguments(kw, status, needle):
    rc, msg = _call("gb_paged_attention", ctypes.byref(_batch()), ctypes.byref(_attn(**kw)), None)
    assert rc == status and needle in msg, (rc, msg)


def test_empty_batches_are_no_ops():
    for kw in (dict(n_seqs=0), dict(total_q=0)):
        assert _call("gb_paged_rope_append", ctypes.byref(_batch(**kw)), ctypes.byref(_rope()), None)[0] == _lib.GB_OK
        assert _call("gb_paged_attention", ctypes.byref(_batch(**kw)), ctypes.byref(_attn()), None)[0] == _lib.GB_OK
    assert _call("gb_sample", ctypes.byref(_sample(rows=0)), None)[0] == _lib.GB_OK
    assert _call("gb_paged_rope_append", None, ctypes.byref(_rope()), None)[0] == INV
    assert _call("gb_paged_attention", ctypes.byref(_batch()), None, None)[0] == INV
    assert _call("gb_sample", None, None)[0] == INV


def test_workspace_size_needs_no_device():
    n = ctypes.c_int64()
    assert _call("gb_paged_attention_workspace", ctypes.byref(_batch()), 4, ctypes.byref(n))[0] == _lib.GB_OK
    assert n.value > 0 and n.value % 256 == 0
    assert _call("gb_paged_attention_workspace", ctypes.byref(_batch()), 5, ctypes.byref(n))[0] == INV
    assert _call("gb_paged_attention_workspace", ctypes.byref(_batch()), 4, None)[0] == INV


@pytest.mark.parametrize("kw,status,needle", [
    (dict(struct_size=1), INV, "struct_size"), (dict(dtype=9), INV, "dtype"), (dict(rows=-1), INV, "rows"),
    (dict(vocab=0), INV, "vocab"), (dict(vocab=400001), UNS, "vocab"), (dict(row_stride=99), INV, "row_stride"),
    (dict(logits_dev=None), INV, "null"), (dict(u_dev=None), INV, "null"), (dict(token_dev=None), INV, "null"),
    (dict(logits_dev=P + 2), INV, "aligned"),
])
def test_sample_refuses_bad_arguments(kw, status, needle):
    rc, msg = _call("gb_sample", ctypes.byref(_sample(**kw)), None)
    assert rc == status and needle in msg, (rc, msg)


@pytest.mark.parametrize("kw,needle", [
    (dict(src=[0], dst=[4]), "dst page"), (dict(src=[0], dst=[-1]), "dst page"), (dict(src=[4], dst=[0]), "src page"),
    (dict(src=[0, 1], dst=[2, 2]), "written twice"), (dict(src=[0, 1], dst=[1, 2]), "both read and written"),
    (dict(src=[0], dst=[0]), "both read and written"), (dict(page_bytes=24), "multiples of 16"),
    (dict(page_stride=32, page_bytes=64), "multiples of 16"), (dict(pool=P + 8), "aligned"), (dict(pool=None), "null"),
    (dict(n_pools=-1), ">= 0"),
])
def test_page_copy_refuses_bad_lists(kw, needle):
    kw = dict(dict(src=[0], dst=[1], page_bytes=64, page_stride=64, pool=P, n_pools=1), **kw)
    n = len(kw["src"])
    i32 = ctypes.c_int32 * n
    pools, src, dst = (ctypes.c_void_p * 1)(kw["pool"]), i32(*kw["src"]), i32(*kw["dst"])
    rc, msg = _call("gb_paged_copy", ctypes.addressof(pools), kw["n_pools"], 4, kw["page_bytes"], kw["page_stride"],
                    ctypes.addressof(src), ctypes.addressof(dst), n, None)
    assert rc == INV and needle in msg, (rc, msg)
    assert _call("gb_paged_copy", None, 0, 4, 64, 64, None, None, 0, None)[0] == _lib.GB_OK


def test_page_pool_against_a_model_of_its_sequences():
    """Random adds, extensions, forks, truncations, frees and compactions: the
    pages hold what each sequence wrote, through the copies it was told of."""
    r = random.Random(3)
    page, n_pages = 4, 40
    pool = paged.PagePool(n_pages, page)
    memory = [[None] * page for _ in range(n_pages)]  # what the device would hold
    model, counter = {}, 0

    def move(src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for a, b in zip(src, dst):
            memory[b] = list(memory[a])

    for _ in range(3000):
        op = r.choice(("add", "extend", "extend", "extend", "fork", "truncate", "free", "compact"))
        seqs = list(model)
        if op == "add" and len(seqs) < 12:
            model[pool.add()] = []
        elif not seqs:
            continue
        elif op == "extend":
            s, n = r.choice(seqs), r.randrange(0, 7)
            before = (pool.pages(s), pool.n_free)
            try:
                move(*pool.extend(s, n))
            except GalliumError as e:
                assert e.status == _lib.GB_ERR_NO_MEMORY and (pool.pages(s), pool.n_free) == before
                pool.free(s)
                del model[s]
                continue
            for _ in range(n):
                counter += 1
                p = len(model[s])
                memory[pool.pages(s)[p // page]][p % page] = counter
                model[s].append(counter)
        elif op == "fork" and len(seqs) < 12:
            s = r.choice(seqs)
            model[pool.fork(s)] = list(model[s])
        elif op == "truncate":
            s = r.choice(seqs)
            n = r.randint(0, len(model[s]))
            pool.truncate(s, n)
            del model[s][n:]
        elif op == "free":
            s = r.choice(seqs)
            pool.free(s)
            del model[s]
        elif op == "compact":
            move(*pool.compact())
            held = {p for s in model for p in pool.pages(s)}
            assert not held or max(held) == len(held) - 1
        held = {p for s in model for p in pool.pages(s)}
        assert pool.n_free == n_pages - len(held)
        for s, want in model.items():
            assert pool.length(s) == len(want)
            pages = pool.pages(s)
            assert [memory[pages[i // page]][i % page] for i in range(len(want))] == want
    t = pool.table(list(model), width=20)
    assert t.dtype == np.int32 and t.shape == (len(model), 20)


def test_page_pool_refusals():
    pool = paged.PagePool(2, 4)
    s = pool.add()
    for call in (lambda: pool.extend(s, -1), lambda: pool.free(99), lambda: pool.truncate(s, 1),
                 lambda: pool.fork(99), lambda: paged.PagePool(0, 4)):
        with pytest.raises(GalliumError) as e:
            call()
        assert e.value.status == INV
    pool.extend(s, 8)
    with pytest.raises(GalliumError):
        pool.table([s], width=1)
    with pytest.raises(GalliumError) as e:
        pool.extend(s, 1)
    assert e.value.status == _lib.GB_ERR_NO_MEMORY


def test_python_refuses_host_tensors():
    import torch

    t = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(GalliumError):
        paged.PagedBatch(t, t[:1], t[None, :1], page_size=16, total_q=1, max_q_len=1, max_kv_len=1)
    with pytest.raises(GalliumError):
        paged.copy_pages(torch.zeros(1, 4, 8), [0], [1])
    with pytest.raises(GalliumError):
        paged.copy_pages([], [0], [])
    from gallium_b200 import sampling
    with pytest.raises(GalliumError):
        sampling.sample(torch.zeros(2, 8), torch.zeros(2))
