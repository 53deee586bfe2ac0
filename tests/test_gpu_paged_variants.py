"""Which attention kernel a batch gets, read from the graph that captures the call."""
import re

import pytest

from gallium_b200 import paged

from test_gpu_paged import Case

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:DEBUG")]


def _kernels(c, tmp_path, **kw):
    """The mangled names of the kernels that an attention call launches."""
    import torch

    batch = c.batch()
    out = torch.empty_like(c.q)
    paged.attention(batch, c.q, c.k, c.v, out=out, **kw)
    graph = torch.cuda.CUDAGraph(keep_graph=True)  # else the dump has nothing to read
    graph.enable_debug_mode()
    with torch.cuda.graph(graph):
        paged.attention(batch, c.q, c.k, c.v, out=out, **kw)
    dot = tmp_path / "graph.dot"
    graph.debug_dump(str(dot))
    return re.findall(r"attn_\w+_kernel\w*", dot.read_text())


@pytest.mark.parametrize("lens,many", [
    ([(1, 60)] * 74 + [(500, 4500)], False),   # one chunk: 256 tiles of many keys, whatever decodes beside it
    ([(1, 60)] * 74 + [(500, 700)], True),     # of few keys
    ([(1, 60)] * 74 + [(100, 2500)], True),    # few tiles
    ([(1, 60)] * 74 + [(350, 2500)], True),
    ([(1, 60)] * 74 + [(100, 4500)], False),
    ([(1, 60)] * 2 + [(1200, 4500)], True),    # 600 tiles of their own
    ([(1200, 9000)], False),                   # of very many keys
    ([(500, 700)], False),
])
def test_small_ctas_for_many_tiles_or_beside_decoding_sequences_of_few_keys(lens, many, tmp_path):
    names = [n for n in _kernels(Case(lens, heads=64, kvh=8, page=64, seed=61), tmp_path) if "tile" in n]
    assert names and all(("Lb1" in n) == many for n in names), names
