"""A bounded wait of the attention kernel for chunks that runs out: GB_ERR_TIMEOUT
from the batch, then a clean call.

With the test hooks the wait limit drops to 50 ms and the first CTA leaves its queries
unread, so the MMA warp waits for them, the softmax warps for its scores and, where the
keys are many, the producer warp for a free slot, until the limit.  Each warp has to
leave its loop as a whole: lanes that left alone would keep the others from ever
meeting them again.  Nothing faults or hangs."""
import time

import pytest

from gallium_b200 import GalliumError, _lib, paged

from test_gpu_paged import MANY, Case


def test_hooks_check_their_arguments():
    lib = _lib.load_library()
    for us in (-1, 10_000_001):
        assert lib.gb_paged_set_test_hooks(us, 0) == _lib.GB_ERR_INVALID_ARG
    assert lib.gb_paged_set_test_hooks(0, 0) == _lib.GB_OK


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(dim=128), dict(dim=256), MANY])
@pytest.mark.parametrize("lens", [[(200, 200), (1, 50)], [(40, 9000)]])
def test_withheld_queries_time_out_and_the_next_call_is_clean(lens, kw):
    import torch

    lib = _lib.load_library()
    c = Case(lens, seed=51, **kw)
    batch = c.batch()
    good = paged.attention(batch, c.q, c.k, c.v, out=torch.zeros_like(c.q))
    batch.check()
    _lib.check(lib.gb_paged_set_test_hooks(50_000, 1))
    try:
        t0 = time.time()
        paged.attention(batch, c.q, c.k, c.v)
        with pytest.raises(GalliumError) as e:
            batch.check()
        assert time.time() - t0 < 5.0
        assert e.value.status == _lib.GB_ERR_TIMEOUT
    finally:
        _lib.check(lib.gb_paged_set_test_hooks(0, 0))
    for _ in range(2):
        assert torch.equal(paged.attention(batch, c.q, c.k, c.v, out=torch.zeros_like(c.q)), good)
    batch.check()
