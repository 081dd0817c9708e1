"""The plain forms that the GPU tests of the routed filter bank compare with, against differences and closed cases."""
import numpy as np
import pytest

import filters as F
import routed_ref as ref


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_route_backward_is_the_derivative(score, renormalise):
    rng = np.random.default_rng(1)
    s = rng.standard_normal((5, 7))
    kw = dict(score=score, renormalise=renormalise, scale=2.5, score_scale=-0.5)
    idx, w, _ = ref.route(s, 3, **kw)
    dw = rng.standard_normal(w.shape)
    got = ref.route_backward(s, idx, dw, **kw)
    h = 1e-6                                  # error of a central difference: h^2 / 6 of a third derivative of order one, and eps / h
    for t in range(5):
        for f in range(7):
            up, dn = s.copy(), s.copy()
            up[t, f] += h
            dn[t, f] -= h
            iu, wu, _ = ref.route(up, 3, **kw)
            id_, wd, _ = ref.route(dn, 3, **kw)
            assert np.array_equal(iu, idx) and np.array_equal(id_, idx)
            assert abs(got[t, f] - (dw * (wu - wd)).sum() / (2 * h)) < 1e-8


def test_route_closed_void_and_ties():
    s = np.array([[1.0, 1.0, 0.0], [-np.inf, 2.0, -np.inf], [-np.inf] * 3, [0.0, np.nan, 1.0], [np.inf, 0.0, 0.0]])
    idx, w, counts = ref.route(s, 2)
    assert idx.tolist() == [[0, 1], [1, -1], [-1, -1], [-1, -1], [-1, -1]]
    assert w[:3].tolist() == [[0.5, 0.5], [1.0, 0.0], [0.0, 0.0]] and np.isnan(w[3:]).all()
    assert counts.tolist() == [1, 2, 0]


def test_pack_is_within_half_a_scale():
    rng = np.random.default_rng(2)
    X = rng.standard_normal((3, 130)) * np.exp(rng.standard_normal((3, 130)))
    q, scales = ref.pack(X)
    d = np.repeat(scales.astype(np.float64), 64, axis=1)[:, :130]
    # half a scale, and the largest value of a block is at most 127 (1 + 2^-24) scales
    assert (np.abs(ref.unpack(q, scales) - X) <= d * (0.5 + 127 * 2.0 ** -24)).all()


@pytest.mark.parametrize("shape", [(8, 1), (4, 8), (1, 1), (1, 8)])
def test_backward_is_the_derivative(oracle, shape):
    rng = np.random.default_rng(3)
    R, C = shape
    X, D = rng.standard_normal((2, R, C)), rng.standard_normal((2, R, C))
    bank = np.stack([F.random_filter(4, s) for s in range(3)])
    idx = np.array([[0, 2], [2, -1]], dtype=np.int32)
    w = rng.standard_normal((2, 2))
    grad, dfilters, dw, dX = ref.backward(oracle, D, X, bank, idx, w)
    h = 1e-6
    cost = lambda X, bank, w: (D * ref.forward(oracle, X, bank, idx, w)).sum()

    def check(got, arg, at):
        up, dn = [X, bank, w], [X, bank, w]
        up[arg], dn[arg] = up[arg].copy(), dn[arg].copy()
        up[arg][at] += h
        dn[arg][at] -= h
        assert abs(got[at] - (cost(*up) - cost(*dn)) / (2 * h)) < 1e-7

    for at in np.ndindex(bank.shape):
        check(dfilters, 1, at)
    for at in np.ndindex(w.shape):
        check(dw, 2, at)
    for at in np.ndindex(X.shape):
        check(dX, 0, at)
    assert np.allclose(grad[0, 1] + grad[1, 0], dfilters[2], atol=1e-12)
