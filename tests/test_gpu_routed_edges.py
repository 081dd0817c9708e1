"""The routed filter bank where values say that there is no answer, lie next to each other, or share memory."""
import numpy as np
import pytest

import routed_ref as ref
from test_gpu_routed import bank_of, run_backward, run_forward

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch
    from wavenet_amd import Context
    c = Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    torch.cuda.synchronize()
    c.close()


# ---- checkpoints that a transform keeps ---------------------------------------------------------------------------

@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 1e300])
@pytest.mark.parametrize("k", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("R,C", [(64, 64), (1024, 1), (16, 32), (2, 1024)])
def test_kept_values_that_are_not_finite_under_several_filters(ctx, R, C, k, value):
    """Every wave of a 64x64 example keeps columns of its own: a value without a scale in any of them reads back as NaN."""
    rng = np.random.default_rng(k)
    n, N = R * C, 4
    at = [0, 4, 8, 12, 16, 20, 63, 31]                      # blocks: columns of a 64x64 example
    B = len(at) + 2
    X = rng.standard_normal((B, n))
    for e, block in enumerate(at):
        X[e, (64 * block + 17 * e + 5) % n] = value
    X[len(at), [3, 64 * 5 % n, n - 1]] = value              # in several blocks; the last example has none
    idx = np.tile(np.arange(k, dtype=np.int32), (B, 1))
    w = rng.standard_normal((B, k))
    bank = bank_of(5, N, 0)
    with np.errstate(invalid="ignore"):
        _, q, sc = run_forward(ctx, np.transpose(X.reshape(B, C, R), (0, 2, 1)), bank, idx, w, keep=True)
    rq, rs = ref.pack(X)
    assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(sc.cpu().numpy(), rs, equal_nan=True)
    back = ref.unpack(q.cpu().numpy(), sc.cpu().numpy())
    assert np.array_equal(back, ref.unpack(rq, rs), equal_nan=True) and np.isnan(back[:-1]).any(axis=1).all()
    assert np.isfinite(back[-1]).all()
    # and so does the gradient at them
    D = rng.standard_normal((B, R, C))
    grad, _, dw, _ = run_backward(ctx, D, bank, idx, w, 5, N, q=q, sc=sc)
    assert np.isnan(dw[:-1]).all() and np.isnan(grad[:-1]).any(axis=2).all()
    assert np.isfinite(dw[-1]).all() and np.isfinite(grad[-1]).all()
