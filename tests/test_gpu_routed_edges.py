"""The routed filter bank where values say that there is no answer, lie next to each other, or share memory."""
import numpy as np
import pytest

import routed_ref as ref
from test_gpu_routed import bank_of, dev, run_backward, run_forward, run_route

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


# ---- router: values next to each other ------------------------------------------------------------------------------

@pytest.mark.parametrize("score_scale", [1.0, -1.0, 0.5])
@pytest.mark.parametrize("F_,k", [(2, 1), (8, 1), (8, 3), (60, 16), (256, 8), (1000, 16)])
def test_route_orders_the_smallest_scores(ctx, F_, k, score_scale):
    """Scores a few units of the smallest 64-bit number apart, of either sign, among zeros, and where normal numbers begin."""
    rng = np.random.default_rng(F_ + k)
    unit = 5e-324
    rows = [rng.integers(-m, m + 1, (12, F_)) * unit for m in (1, 3, 40, 1023, 2050, 5000)]
    rows.append((2 ** 52 + rng.integers(-1500, 1500, (12, F_))) * unit)
    rows.append(-(2 ** 53 + rng.integers(0, 1500, (12, F_))) * unit)
    zeros = np.zeros((4, F_))
    zeros[0, -1], zeros[1, -1], zeros[2, 0], zeros[3, F_ // 2] = 1e-321, unit, -unit, 1022 * unit
    s = np.concatenate(rows + [zeros])
    for kw in (dict(), dict(score="sigmoid"), dict(groups=2, groups_kept=1, renormalise=False)):
        idx, w, counts = run_route(ctx, dev(s), k, score_scale=score_scale, **kw)
        ri, rw, rc = ref.route(s, k, score_scale=score_scale, **kw)
        assert np.array_equal(idx, ri) and np.array_equal(counts, rc)
        assert np.allclose(w, rw, rtol=2000 * 2.0 ** -53, atol=0)
