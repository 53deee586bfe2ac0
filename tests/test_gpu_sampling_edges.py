"""gb_sample at the ends of its settings, against the definition in float64."""
import numpy as np
import pytest

from test_gpu_sampling import _check, _rows, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1e-38, 9e-38, 1.1e-37, 3e-37])
@pytest.mark.parametrize("kw", [dict(k=50), dict(least=1.0), dict(k=50, least=0.5), dict(k=50, p=0.6), dict(p=0.6),
                                dict(k=600, p=0.6, least=0.1)])
def test_tiny_temperatures(t, kw):
    """Temperatures whose reciprocal times 32 no longer fits in f32, with a largest logit
    of 0 and of other sizes, alone and among many equals: every row is written."""
    import torch

    rng = np.random.default_rng(3)
    x = -_rows(8, 1000, seed=4).abs()
    x[:, 77] = 0.0
    x[1] = 0.0
    x[2, ::3] = 0.0
    x[3] += 5.0
    x[4] -= 5.0
    x[5, ::7] = 0.0
    x[6, 500:] = float("-inf")
    x[7] *= 1e-37
    n = x.shape[0]
    _check(x, rng.random(n), t=[t] * n, **{k: [v] * n for k, v in kw.items()})
    # nothing is left of what the outputs held
    tok, lp = (torch.full((n,), v, dtype=d, device="cuda") for v, d in ((-7, torch.int32), (7.0, torch.float32)))
    _run(x, rng.random(n), [t] * n, **{k: [v] * n for k, v in kw.items()}, tokens=tok, logprobs=lp)
    assert (tok >= 0).all() and (lp <= 0).all()
