"""The routed filter bank on a real MI355X against the plain 64-bit forms of routed_ref.py."""
import numpy as np
import pytest

import filters as F
import routed_ref as ref

pytestmark = pytest.mark.gpu

TYPES = ["f64", "f32", "f16", "bf16"]
HALF_STEP = {"f64": 2.0 ** -53, "f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# a transform's value passes at most 2 * 12 levels of at most 32 multiply-adds, 768 roundings of 2^-53, each carried on with
# a gain of at most about 20 relative to the largest value (tap sums of 1.9 against norms of 1.41 over ten levels): 1.7e-12
TOL = 1e-11


def torch_type(t):
    import torch
    return {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


@pytest.fixture(scope="module")
def ctx():
    import torch
    from wavenet_amd import Context
    c = Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    torch.cuda.synchronize()
    c.close()


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def full(shape, value, dtype):
    import torch
    return torch.full(shape, value, dtype=dtype, device="cuda")


def host(t):
    import torch
    return t.to(torch.float64).cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def laid_out(scores, layout):
    """A device matrix of the scores: dense rows, filter by filter, or rows and filters with gaps."""
    import torch
    T, F_ = scores.shape
    if layout == "rows":
        return scores.contiguous()
    if layout == "filters":
        return scores.t().contiguous().t()
    big = torch.full((T, 2 * F_ + 3), float("nan"), dtype=scores.dtype, device=scores.device)
    view = big[:, 1:2 * F_ + 1:2]
    view.copy_(scores)
    return view


def run_route(ctx, s, k, counts=True, **kw):
    import torch
    T, F_ = s.shape
    idx, w = full((T + 1, k), -7, torch.int32), full((T + 1, k), 7.0, torch.float64)
    cnt = full((F_ + 1,), -7, torch.int32) if counts else None
    ctx.route(s, T, F_, idx, w, k=k, row_stride=s.stride(0), col_stride=s.stride(1), counts=cnt, **kw)
    torch.cuda.synchronize()
    assert (idx[T] == -7).all() and (w[T] == 7.0).all() and (cnt is None or cnt[F_] == -7)
    return idx[:T].cpu().numpy(), w[:T].cpu().numpy(), None if cnt is None else cnt[:F_].cpu().numpy()


ROUTINGS = [
    # T, F, k, options
    (1, 8, 2, dict()),
    (1, 1, 1, dict(score="sigmoid", renormalise=False)),
    (3, 2, 2, dict(scale=2.5)),
    (17, 16, 16, dict(renormalise=False)),
    (33, 17, 5, dict(score="sigmoid", bias=True)),
    (130, 33, 3, dict(bias=True, score_scale=-8.0)),
    (61, 64, 6, dict(groups=8, groups_kept=4, score="sigmoid", bias=True, scale=2.5)),
    (61, 60, 4, dict(groups=5, groups_kept=2, renormalise=False)),
    (19, 100, 7, dict(groups=20, groups_kept=3, bias=True)),
    (300, 128, 8, dict(score="sigmoid", renormalise=False, score_scale=0.5)),
    (29, 256, 8, dict(groups=64, groups_kept=9, score="sigmoid")),
    (9, 257, 1, dict(bias=True)),
    (5, 512, 16, dict(groups=4, groups_kept=1, bias=True)),
    (7, 1000, 9, dict(renormalise=False, bias=True)),
    (4, 1024, 16, dict(score="sigmoid", groups=2, groups_kept=1)),
    (5000, 12, 2, dict(score="sigmoid", bias=True)),
]


@pytest.mark.parametrize("layout", ["rows", "filters", "gaps"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,F_,k,opt", ROUTINGS)
def test_route(ctx, T, F_, k, opt, dtype, layout):
    rng = np.random.default_rng(T + 13 * F_ + k)
    opt = dict(opt)
    s = laid_out(dev(rng.standard_normal((T, F_)) * 1.5, torch_type(dtype)), layout)
    bias = rng.standard_normal(F_) * 0.05 if opt.pop("bias", False) else None
    idx, w, counts = run_route(ctx, s, k, bias=None if bias is None else dev(bias), **opt)
    ri, rw, rc = ref.route(host(s), k, bias=bias, **opt)
    assert np.array_equal(idx, ri) and np.array_equal(counts, rc)
    # exponentials of |s| < 100: 100 * 2^-53 from the argument, a few 2^-53 from exp, F * 2^-53 from the sum
    assert np.allclose(w, rw, rtol=2000 * 2.0 ** -53, atol=0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_masks_and_values_without_an_answer(ctx, score, renormalise, groups, kept, biased):
    inf, nan, low = np.inf, np.nan, -np.finfo(np.float64).max
    rows = [[0, 1, 2, 3, 4, 5, 6, 7], [-inf] * 8, [-inf] * 3 + [0.5] + [-inf] * 4, [low] * 8, [low] * 7 + [0], [-inf, low] * 4,
            [nan] + [0] * 7, [0] * 7 + [nan], [-inf] * 7 + [nan], [inf] + [0] * 7, [3] * 8, [0, -0.0] * 4, [-800] * 4 + [-900] * 4,
            [800] * 2 + [-800] * 6, [1e-310] * 8, [-inf, 1, -inf, 2, -inf, -inf, -inf, -inf]]
    s = np.array(rows, dtype=np.float64)
    bias = np.array([0, 0.1, 0, -inf, 0, nan, 0, inf]) if biased else None
    kw = dict(score=score, renormalise=renormalise, groups=groups, groups_kept=kept)
    idx, w, counts = run_route(ctx, dev(s), 3, bias=None if bias is None else dev(bias), **kw)
    ri, rw, rc = ref.route(s, 3, bias=bias, **kw)
    assert np.array_equal(idx, ri) and np.array_equal(counts, rc)
    assert np.allclose(w, rw, rtol=2000 * 2.0 ** -53, atol=0, equal_nan=True)


def test_route_equal_scores_go_to_the_lowest_filter(ctx):
    rng = np.random.default_rng(5)
    s = rng.integers(0, 3, (200, 200)).astype(np.float64)          # ties everywhere
    for kw in (dict(), dict(groups=10, groups_kept=3), dict(score="sigmoid", bias=np.zeros(200))):
        opt = {k: (dev(v) if k == "bias" else v) for k, v in kw.items()}
        idx, _, _ = run_route(ctx, dev(s), 10, **opt)
        assert np.array_equal(idx, ref.route(s, 10, **kw)[0])


def test_route_values_closer_than_floats(ctx):
    """Shares that differ by less than a float's step, and a bias that decides between them."""
    rng = np.random.default_rng(6)
    base = rng.standard_normal((64, 1))
    step = rng.permuted(np.tile(np.arange(40), (64, 1)), axis=1)
    s = base + step * 1e-12
    # The share of step m is p0 (1 + m 1e-12 + O(1e-22)), the score of a group p0 (2 + (m1 + m2) 1e-12 + O(1e-22)) from its two
    # largest steps: groups of equal m1 + m2 differ by 1e-22, which 64 bits (1e-16) do not tell apart whatever the order of
    # the sums, so rows whose second and third group have equal sums have no one answer.
    sums = np.sort(np.sort(step.reshape(64, 4, 10), axis=2)[:, :, -2:].sum(axis=2), axis=1)
    decided = sums[:, 2] != sums[:, 1]
    assert decided.sum() > 50
    for kw in (dict(), dict(bias=np.zeros(40)), dict(bias=np.zeros(40), score="sigmoid"), dict(groups=4, groups_kept=2, bias=np.zeros(40))):
        opt = {k: (dev(v) if k == "bias" else v) for k, v in kw.items()}
        idx, _, _ = run_route(ctx, dev(s), 8, **opt)
        rows = decided if "groups" in kw else slice(None)
        assert np.array_equal(idx[rows], ref.route(s, 8, **kw)[0][rows])


@pytest.mark.parametrize("layout", ["rows", "filters", "gaps"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,F_,k,opt", ROUTINGS)
def test_route_backward(ctx, T, F_, k, opt, dtype, layout):
    import torch
    rng = np.random.default_rng(T + 13 * F_ + k)
    opt = {a: b for a, b in opt.items() if a != "bias"}
    s = laid_out(dev(rng.standard_normal((T, F_)) * 1.5, torch_type(dtype)), layout)
    idx = ref.route(host(s), k, **opt)[0]
    idx[T // 2, 0] = -1                                            # nothing there
    idx[T // 3, k - 1] = F_                                        # beyond the filters
    dw = rng.standard_normal((T, k))
    ds = laid_out(full((T, F_), float("nan"), torch_type(dtype)), layout)
    ctx.route_backward(s, T, F_, dev(idx), dev(dw), ds, k=k, row_stride=s.stride(0), col_stride=s.stride(1), **opt)
    torch.cuda.synchronize()
    few = {a: b for a, b in opt.items() if a not in ("groups", "groups_kept")}
    want = ref.route_backward(host(s), idx, dw, **few)
    # differences of products of order one, computed to 2000 * 2^-53 of their parts, rounded once; fp16 has steps of 2^-24
    # below 2^-14
    bound = HALF_STEP[dtype] * np.abs(want) + 1e-11 * max(1.0, np.abs(want).max()) + (2.0 ** -25 if dtype == "f16" else 0)
    assert (np.abs(host(ds) - want) <= bound).all()
    if layout == "gaps":                                           # what lies between the rows is left alone
        base = ds._base if ds._base is not None else ds
        assert torch.isnan(base[:, 0]).all() and torch.isnan(base[:, 2::2]).all()


def test_route_backward_in_place_and_against_differences(ctx):
    import torch
    rng = np.random.default_rng(8)
    T, F_, k, h = 40, 11, 3, 1e-6
    for kw in (dict(), dict(renormalise=False), dict(score="sigmoid"), dict(score="sigmoid", renormalise=False)):
        s = rng.standard_normal((T, F_))
        idx, w, _ = run_route(ctx, dev(s), k, **kw)
        dw = rng.standard_normal((T, k))
        g = dev(s)
        ctx.route_backward(g, T, F_, dev(idx), dev(dw), g, k=k, **kw)
        torch.cuda.synchronize()
        for f in range(F_):
            up, dn = s.copy(), s.copy()
            up[:, f] += h
            dn[:, f] -= h
            iu, wu, _ = run_route(ctx, dev(up), k, **kw)
            il, wl, _ = run_route(ctx, dev(dn), k, **kw)
            same = (iu == il).all(axis=1) & (iu == idx).all(axis=1)
            assert same.mean() > 0.9
            assert np.abs((dw * (wu - wl)).sum(axis=1) / (2 * h) - g.cpu().numpy()[:, f])[same].max() < 1e-8


# ---- checkpoints ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,n,gap", [(1, 1, 0), (3, 2, 0), (5, 63, 1), (2, 64, 0), (4, 65, 0), (7, 128, 3), (37, 777, 0), (2, 1000, 24),
                                     (300, 256, 0), (3, 4096, 0), (1, 100003, 0)])
def test_checkpoint(ctx, B, n, gap, dtype):
    import torch
    rng = np.random.default_rng(B + n)
    tt = torch_type(dtype)
    x = rng.standard_normal((B, n)) * np.exp(rng.standard_normal((B, n)))
    x[0, : n // 3] = 0.0                                           # whole blocks of nothing among them
    wide = full((B, n + gap), float("nan"), tt)
    wide[:, :n] = dev(x).to(tt)
    nb = -(-n // 64)
    q, sc = full((B * n + 1,), 77, torch.int8), full((B * nb + 1,), 77.0, torch.float32)
    ctx.checkpoint_pack(wide, B, n, q, sc, row_stride=n + gap)
    back = full((B, n + gap), float("nan"), tt)
    ctx.checkpoint_unpack(q, sc, B, n, back, row_stride=n + gap)
    torch.cuda.synchronize()
    assert q[-1] == 77 and sc[-1] == 77.0 and (gap == 0 or torch.isnan(back[:, n:]).all())
    rq, rs = ref.pack(host(wide[:, :n]))
    assert np.array_equal(q[:-1].cpu().numpy().reshape(B, n), rq)
    assert np.array_equal(sc[:-1].cpu().numpy().reshape(B, nb), rs)
    want = ref.unpack(rq, rs)
    tiny = {"f16": 2.0 ** -25, "f32": 2.0 ** -150}.get(dtype, 0.0)
    got = host(back[:, :n])
    if dtype in ("f64", "f32"):
        assert np.array_equal(got, want.astype(np.float64 if dtype == "f64" else np.float32))
    assert (np.abs(got - want) <= HALF_STEP[dtype] * np.abs(want) + tiny).all()


def test_checkpoint_values_without_a_scale(ctx):
    import torch
    big = np.finfo(np.float64).max
    rows = np.zeros((9, 130))
    rows[0, 5] = np.nan
    rows[1, 70] = np.inf
    rows[2, 129] = -np.inf
    rows[3, 3] = big
    rows[4, :64] = 1e39 * np.linspace(-1, 1, 64)
    rows[5, :] = 1e-320
    rows[6, :] = np.linspace(-1, 1, 130) * 1e-40
    rows[7, :64] = np.linspace(-1, 1, 64) * 5e40                    # beyond 127 times the largest float
    rows[8, :] = -1.0
    x = dev(rows)
    q, sc, back = full((9, 130), 7, torch.int8), full((9, 3), 7.0, torch.float32), torch.empty_like(x)
    ctx.checkpoint_pack(x, 9, 130, q, sc)
    ctx.checkpoint_unpack(q, sc, 9, 130, back)
    torch.cuda.synchronize()
    rq, rs = ref.pack(rows)
    assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(sc.cpu().numpy(), rs, equal_nan=True)
    got = back.cpu().numpy()
    assert np.array_equal(got, ref.unpack(rq, rs), equal_nan=True)
    assert np.isnan(got[0, :64]).all() and (got[0, 64:] == 0).all() and np.isnan(got[3, :64]).all() and np.isnan(got[7, :64]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_checkpoint_reads_back_rounded_once(ctx, dtype):
    """Scales for which the nearest float of a value lies on a border of the 16-bit type and the value does not."""
    import torch
    tt = torch_type(dtype)
    rng = np.random.default_rng(3)
    sc = np.abs(rng.standard_normal((4000, 1))).astype(np.float32) + np.float32(0.01)
    bits = 13 if dtype == "f16" else 16
    sc = (sc.view(np.uint32) & ~np.uint32((1 << bits) - 1) | np.uint32(1 << (bits - 1))).view(np.float32)   # halfway values
    sc[1::2] = np.nextafter(sc[1::2], np.float32(9))
    q = rng.integers(-127, 128, (4000, 64)).astype(np.int8)
    back = full((4000, 64), 0, tt)
    ctx.checkpoint_unpack(dev(q), dev(sc), 4000, 64, back)
    torch.cuda.synchronize()
    v = ref.unpack(q, sc)
    got = host(back)
    # the nearest value of the type: no neighbour is nearer
    for neighbour in (torch.nextafter(back, full((), float("inf"), tt)), torch.nextafter(back, full((), -float("inf"), tt))):
        assert (np.abs(got - v) <= np.abs(host(neighbour) - v)).all()


# ---- transforms -------------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (2, 1), (1, 2), (2, 2), (8, 1), (1, 8), (8, 8), (32, 8), (64, 1), (1, 64), (128, 1), (256, 1), (512, 1), (16, 32),
          (1024, 1), (1, 1024), (32, 64), (2048, 1), (64, 64), (4096, 1), (2, 1024), (128, 32)]


def bank_of(F_, N, seed):
    base = F.daubechies(N) if N <= 16 else None
    return np.stack([F.perturbed(base, 1e-2, seed + i) if base is not None else F.random_filter(N, seed + i) for i in range(F_)])


def flat(X):
    """[B, R, C] -> [B, n] column-major on the device"""
    return dev(np.ascontiguousarray(np.transpose(X, (0, 2, 1))).reshape(len(X), -1))


def unflat(t, R, C):
    a = t.cpu().numpy()
    return np.transpose(a.reshape(len(a), C, R), (0, 2, 1))


def near(got, want, tol=TOL):
    scale = np.abs(want).max() if want.size else 0.0
    return (np.abs(got - want) <= tol * max(scale, 1e-300)).all()


def entries(rng, B, F_, k):
    """Filters in any order, one twice in an example, one example without any, indices that name none."""
    idx = rng.integers(0, F_, (B, k)).astype(np.int32)
    w = rng.standard_normal((B, k))
    if B > 2:
        idx[1, :] = idx[1, 0]
        idx[2, :] = -1
    if B > 3:
        idx[3, -1] = F_
        w[3, 0] = 0.0
    if B > 4:
        idx[4, 0] = -2 ** 31
    return idx, w


def run_forward(ctx, X, bank, idx, w, keep, k=None):
    import torch
    B, R, C = X.shape
    n, nb = R * C, -(-R * C // 64)
    Y = full((B * n + 1,), 9.0, torch.float64)
    q, sc = (full((B * n + 1,), 77, torch.int8), full((B * nb + 1,), 77.0, torch.float32)) if keep else (None, None)
    ctx.forward_routed(flat(X), B, R, C, None if bank is None else dev(bank), None if idx is None else dev(idx),
                       None if w is None else dev(w), Y, k=k, q=q, scales=sc)
    torch.cuda.synchronize()
    assert Y[-1] == 9.0
    if keep:
        assert q[-1] == 77 and sc[-1] == 77.0
        q, sc = q[:-1].reshape(B, n), sc[:-1].reshape(B, nb)
    return unflat(Y[:-1].reshape(B, n), R, C), q, sc


def run_backward(ctx, D, bank, idx, w, F_, N, X=None, q=None, sc=None, k=None):
    import torch
    B, R, C = D.shape
    n = R * C
    k = idx.shape[1] if idx is not None else 1
    grad, dw = full((B * k * N + 1,), 9.0, torch.float64), full((B * k + 1,), 9.0, torch.float64)
    dX, dF = full((B * n + 1,), 9.0, torch.float64), full((F_ * N + 1,), 9.0, torch.float64)
    ctx.backprop_routed(flat(D), B, R, C, None if bank is None else dev(bank), None if idx is None else dev(idx),
                        None if w is None else dev(w), grad, X=None if X is None else flat(X), q=q, scales=sc, dfilters=dF, dw=dw, dX=dX)
    torch.cuda.synchronize()
    assert grad[-1] == 9.0 and dw[-1] == 9.0 and dX[-1] == 9.0 and dF[-1] == 9.0
    return (grad[:-1].cpu().numpy().reshape(B, k, N), dF[:-1].cpu().numpy().reshape(F_, N), dw[:-1].cpu().numpy().reshape(B, k),
            unflat(dX[:-1].reshape(B, n), R, C))


@pytest.mark.parametrize("N", [2, 4, 6, 8, 10, 16, 32])
@pytest.mark.parametrize("R,C", SHAPES)
def test_forward_routed(ctx, oracle, R, C, N):
    rng = np.random.default_rng(R + 7 * C + N)
    B, F_, k = 9, 5, 1 + (R + N) % 4
    X = rng.standard_normal((B, R, C))
    bank = bank_of(F_, N, 40)
    idx, w = entries(rng, B, F_, k)
    Y, q, sc = run_forward(ctx, X, bank, idx, w, keep=True)
    assert near(Y, ref.forward(oracle, X, bank, idx, w))
    rq, rs = ref.pack(np.transpose(X, (0, 2, 1)).reshape(B, -1))
    assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(sc.cpu().numpy(), rs)
    assert np.array_equal(run_forward(ctx, X, bank, idx, w, keep=False)[0], Y)


@pytest.mark.parametrize("N", [2, 4, 6, 8, 10, 16, 32])
@pytest.mark.parametrize("R,C", SHAPES)
def test_backprop_routed(ctx, oracle, R, C, N):
    import torch
    rng = np.random.default_rng(R + 7 * C + N)
    B, F_, k = 9, 5, 1 + (R + N) % 4
    X, D = rng.standard_normal((B, R, C)), rng.standard_normal((B, R, C))
    bank = bank_of(F_, N, 40)
    idx, w = entries(rng, B, F_, k)
    got = run_backward(ctx, D, bank, idx, w, F_, N, X=X)
    want = ref.backward(oracle, D, X, bank, idx, w)
    for g, r in zip(got, want):
        assert near(g, r, 1e-10)                    # sums of up to 4096 products of such values
    # from the checkpoint: the gradient at the values that it stands for
    rq, rs = ref.pack(np.transpose(X, (0, 2, 1)).reshape(B, -1))
    Xq = np.transpose(ref.unpack(rq, rs).reshape(B, C, R), (0, 2, 1))
    got_q = run_backward(ctx, D, bank, idx, w, F_, N, q=dev(rq), sc=dev(rs))
    for g, r in zip(got_q, ref.backward(oracle, D, Xq, bank, idx, w)):
        assert near(g, r, 1e-10)
    # the same bits again, and without the outputs that may be left out
    again = run_backward(ctx, D, bank, idx, w, F_, N, q=dev(rq), sc=dev(rs))
    assert all(np.array_equal(a, b) for a, b in zip(got_q, again))
    grad = full((B, k, N), 9.0, torch.float64)
    ctx.backprop_routed(flat(D), B, R, C, dev(bank), dev(idx), dev(w), grad, q=dev(rq), scales=dev(rs))
    torch.cuda.synchronize()
    assert np.array_equal(grad.cpu().numpy(), got_q[0])


@pytest.mark.parametrize("R,C", [(64, 64), (1024, 1), (256, 1), (16, 32)])
@pytest.mark.parametrize("B,F_,k", [(1, 1, 1), (1, 3, 16), (1, 8, 2), (300, 3, 2), (1100, 40, 1)])
def test_routed_batches(ctx, oracle, R, C, B, F_, k):
    """From one example to more than the chip holds at once."""
    rng = np.random.default_rng(B)
    N = 4
    X, D = rng.standard_normal((B, R, C)), rng.standard_normal((B, R, C))
    bank = bank_of(F_, N, 3)
    idx, w = entries(rng, B, F_, k)
    assert near(run_forward(ctx, X, bank, idx, w, keep=False)[0], ref.forward(oracle, X, bank, idx, w))
    for g, r in zip(run_backward(ctx, D, bank, idx, w, F_, N, X=X), ref.backward(oracle, D, X, bank, idx, w)):
        assert near(g, r, 1e-10)


@pytest.mark.parametrize("R,C", [(64, 64), (1024, 1), (8, 8)])
def test_the_contexts_own_filter(ctx, oracle, R, C):
    """Without a bank: what wn_forward and wn_backprop compute, with an 8-bit checkpoint in place of their activations."""
    rng = np.random.default_rng(4)
    a = bank_of(1, 6, 9)
    ctx.set_filter(a[0])
    X, D = rng.standard_normal((5, R, C)), rng.standard_normal((5, R, C))
    Y, q, sc = run_forward(ctx, X, None, None, None, keep=True)
    zero, one = np.zeros((5, 1), dtype=np.int32), np.ones((5, 1))
    assert near(Y, ref.forward(oracle, X, a, zero, one))
    Xq = np.transpose(ref.unpack(q.cpu().numpy(), sc.cpu().numpy()).reshape(5, C, R), (0, 2, 1))
    for g, r in zip(run_backward(ctx, D, None, None, None, 1, 6, q=q, sc=sc), ref.backward(oracle, D, Xq, a, zero, one)):
        assert near(g, r, 1e-10)


@pytest.mark.parametrize("R,C", [(64, 64), (1024, 1), (16, 32), (1, 1)])
def test_weights_without_an_answer_reach_the_result(ctx, R, C):
    rng = np.random.default_rng(4)
    X = rng.standard_normal((4, R, C))
    idx = np.array([[0, 1], [-1, -1], [-1, 0], [1, 0]], dtype=np.int32)
    w = np.array([[0.5, 0.5], [np.nan, np.nan], [np.nan, 1.0], [np.nan, 1.0]])
    Y = run_forward(ctx, X, bank_of(2, 4, 1), idx, w, keep=False)[0]
    assert np.isfinite(Y[0]).all() and np.isnan(Y[1:]).all()
    dX = run_backward(ctx, X, bank_of(2, 4, 1), idx, w, 2, 4, X=X)[3]
    assert np.isfinite(dX[0]).all() and np.isnan(dX[1:]).all()


def test_nothing_to_do(ctx):
    import torch
    e64, e32 = torch.empty(0, dtype=torch.float64, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    counts, dF = full((3,), 5, torch.int32), full((3, 4), 5.0, torch.float64)
    ctx.route(e64, 0, 3, e32, e64, k=2, counts=counts)
    ctx.route_backward(e64, 0, 3, e32, e64, e64, k=2)
    ctx.forward_routed(e64, 0, 64, 64, dev(bank_of(3, 4, 0)), e32, e64, e64, k=2)
    ctx.backprop_routed(e64, 0, 64, 64, dev(bank_of(3, 4, 0)), e32, e64, e64, X=e64, dfilters=dF, k=2)
    ctx.checkpoint_pack(e64, 0, 5, e32.to(torch.int8), e64.float())
    ctx.checkpoint_pack(e64, 5, 0, e32.to(torch.int8), e64.float())
    torch.cuda.synchronize()
    assert (counts == 0).all() and (dF == 0).all()


def test_refusals(ctx):
    import torch
    from wavenet_amd import capi
    E = capi.WavenetError
    s, idx, w = full((4, 8), 0.0, torch.float64), full((4, 2), 0, torch.int32), full((4, 2), 0.0, torch.float64)

    def refused(status, fn, *a, **kw):
        with pytest.raises(E) as err:
            fn(*a, **kw)
        assert err.value.status == status and str(err.value)

    for kw in (dict(k=0), dict(k=9), dict(k=2, groups=3), dict(k=2, groups=4, groups_kept=5), dict(k=2, groups=4, groups_kept=0),
               dict(k=2, groups=0), dict(k=2, scale=float("nan")), dict(k=2, score_scale=0.0), dict(k=2, score_scale=float("inf")), dict(k=2, score=7)):
        refused(capi.WN_ERR_ARG, ctx.route, s, 4, 8, idx.data_ptr(), w.data_ptr(), **kw)
        refused(capi.WN_ERR_ARG, ctx.route_backward, s, 4, 8, idx.data_ptr(), w.data_ptr(), s, **kw)
    for strides in (dict(row_stride=4), dict(row_stride=7), dict(row_stride=0), dict(row_stride=-8), dict(row_stride=1, col_stride=3)):
        refused(capi.WN_ERR_ARG, ctx.route, s, 4, 8, idx.data_ptr(), w.data_ptr(), k=2, **strides)
    refused(capi.WN_ERR_UNSUPPORTED, ctx.route, s.data_ptr(), 4, 1025, idx.data_ptr(), w.data_ptr(), k=2)
    refused(capi.WN_ERR_UNSUPPORTED, ctx.route, s.data_ptr(), 1, 32, idx.data_ptr(), w.data_ptr(), k=17)
    refused(capi.WN_ERR_UNSUPPORTED, ctx.route, s.data_ptr(), 1, 130, idx.data_ptr(), w.data_ptr(), k=1, groups=65, groups_kept=2)
    refused(capi.WN_ERR_ARG, ctx.route, s.data_ptr(), -1, 8, idx.data_ptr(), w.data_ptr(), k=2)
    refused(capi.WN_ERR_ARG, ctx.route, s.data_ptr() + 4, 4, 8, idx.data_ptr(), w.data_ptr(), k=2)
    refused(capi.WN_ERR_ARG, ctx.route, s.data_ptr(), 4, 8, idx.data_ptr(), w.data_ptr(), k=2, dtype=9)
    refused(capi.WN_ERR_ARG, ctx.route, s, 4, 8, None, w, k=2)
    with pytest.raises(ValueError):
        ctx.route(s, 4, 8, idx, w, k=3)                            # too small for three
    with pytest.raises(ValueError):
        ctx.route(s.cpu(), 4, 8, idx, w, k=2)
    with pytest.raises(ValueError):
        ctx.route(s, 5, 8, idx, w, k=1)                            # the scores end before
    with pytest.raises(ValueError):
        ctx.route(s, 4, 8, idx.long(), w, k=2)
    with pytest.raises(ValueError):
        ctx.route(s.long(), 4, 8, idx, w, k=2)
    with pytest.raises(ValueError):
        ctx.route_backward(s, 4, 8, idx, w, s.float(), k=2)

    x, q, sc = full((4, 100), 0.0, torch.float64), full((4, 100), 0, torch.int8), full((4, 2), 0.0, torch.float32)
    refused(capi.WN_ERR_ARG, ctx.checkpoint_pack, x, 4, 100, q, sc, row_stride=99)
    refused(capi.WN_ERR_ARG, ctx.checkpoint_pack, x.data_ptr(), -4, 100, q.data_ptr(), sc.data_ptr())
    refused(capi.WN_ERR_ARG, ctx.checkpoint_unpack, None, sc, 4, 100, x)
    refused(capi.WN_ERR_ARG, ctx.checkpoint_unpack, q.data_ptr(), sc.data_ptr() + 1, 4, 100, x.data_ptr())
    with pytest.raises(ValueError):
        ctx.checkpoint_pack(x, 4, 100, q, sc[:, :1].contiguous())

    X, Y, bank = full((4, 64), 0.0, torch.float64), full((4, 64), 0.0, torch.float64), dev(bank_of(3, 4, 0))
    p = [t.data_ptr() for t in (X, bank, idx, w, Y)]

    def fwd(R=8, C=8, F_=3, N=4, k=2, B=4, idx=p[2], filters=p[1], X=p[0], Y=p[4], **kw):
        ctx.forward_routed(X, B, R, C, filters, idx, p[3], Y, k=k, F=F_, N=N, **kw)

    refused(capi.WN_ERR_BAD_SHAPE, fwd, R=6)
    refused(capi.WN_ERR_BAD_SHAPE, fwd, C=0)
    refused(capi.WN_ERR_BAD_FILTER, fwd, N=3)
    refused(capi.WN_ERR_BAD_FILTER, fwd, N=0)
    refused(capi.WN_ERR_UNSUPPORTED, fwd, N=34)
    refused(capi.WN_ERR_UNSUPPORTED, fwd, R=128, C=64)
    refused(capi.WN_ERR_ARG, fwd, k=0)
    refused(capi.WN_ERR_ARG, fwd, k=17)
    refused(capi.WN_ERR_ARG, fwd, F_=0)
    refused(capi.WN_ERR_ARG, fwd, B=-1)
    refused(capi.WN_ERR_ARG, fwd, idx=None)
    refused(capi.WN_ERR_ARG, fwd, X=None)
    refused(capi.WN_ERR_ARG, fwd, X=p[0] + 4)
    refused(capi.WN_ERR_ARG, fwd, q=q)
    fresh = capi.Context(0)
    with pytest.raises(E) as err:
        fresh.forward_routed(X, 4, 8, 8, None, None, None, Y, F=1, N=4)
    assert err.value.status == capi.WN_ERR_STATE
    fresh.close()
    grad = full((4, 2, 4), 0.0, torch.float64)
    refused(capi.WN_ERR_ARG, ctx.backprop_routed, X, 4, 8, 8, bank, idx, w, grad)                      # neither input
    refused(capi.WN_ERR_ARG, ctx.backprop_routed, X, 4, 8, 8, bank, idx, w, grad, X=X, q=q, scales=sc)  # both
    refused(capi.WN_ERR_ARG, ctx.backprop_routed, X, 4, 8, 8, bank, idx, w, None, X=X)
    with pytest.raises(ValueError):
        ctx.forward_routed(X, 4, 8, 8, bank.float(), idx, w, Y)
    assert capi.load_library().wn_route(None, None, 0, 0, 0, 0, 0, None, None, None, None, None) == capi.WN_ERR_ARG
    assert capi.load_library().wn_forward_routed(None, None, 0, 0, 0, None, 0, 0, None, None, 0, None, None, None) == capi.WN_ERR_ARG


# ---- together ---------------------------------------------------------------------------------------------------

class Mixture:
    """A training pass of a bank: route, transform, sparsity cost, and everything backwards."""

    def __init__(self, ctx, B, R, C, N, F_, k, seed, score="sigmoid"):
        import torch
        rng = np.random.default_rng(seed)
        self.ctx, self.shape, self.k, self.kw = ctx, (B, R, C), k, dict(k=k, score=score)
        n, nb, z = R * C, -(-R * C // 64), lambda *s: full(s, float("nan"), torch.float64)
        self.X, self.bank = flat(rng.random((B, R, C))), dev(bank_of(F_, N, seed))
        self.scores, self.bias = dev(rng.standard_normal((B, F_)).astype(np.float32)), dev(rng.standard_normal(F_) * 0.01)
        self.idx, self.counts = full((B, k), -7, torch.int32), full((F_,), -7, torch.int32)
        self.w, self.Y, self.D, self.S = z(B, k), z(B, n), z(B, n), z(B)
        self.q, self.sc = full((B, n), 0, torch.int8), full((B, nb), 0.0, torch.float32)
        self.grad, self.dF, self.dw, self.dX = z(B, k, N), z(F_, N), z(B, k), z(B, n)
        self.ds = torch.full_like(self.scores, float("nan"))

    def step(self):
        ctx, (B, R, C) = self.ctx, self.shape
        F_ = len(self.bank)
        ctx.route(self.scores, B, F_, self.idx, self.w, bias=self.bias, counts=self.counts, **self.kw)
        ctx.forward_routed(self.X, B, R, C, self.bank, self.idx, self.w, self.Y, q=self.q, scales=self.sc)
        ctx.sparse_term_deriv(self.Y, B, R * C, self.D, self.S)
        ctx.backprop_routed(self.D, B, R, C, self.bank, self.idx, self.w, self.grad, q=self.q, scales=self.sc, dfilters=self.dF,
                            dw=self.dw, dX=self.dX)
        ctx.route_backward(self.scores, B, F_, self.idx, self.dw, self.ds, **self.kw)

    def results(self):
        return [t.cpu().numpy().copy() for t in (self.idx, self.counts, self.w, self.Y, self.S, self.q, self.sc, self.grad, self.dF, self.dw,
                                                 self.dX, self.ds)]


@pytest.mark.parametrize("R,C,N,k", [(64, 64, 4, 2), (16, 32, 8, 3), (256, 1, 6, 1)])
def test_training_pass_of_a_bank(ctx, oracle, R, C, N, k):
    import torch
    m = Mixture(ctx, 23, R, C, N, 7, k, 5)
    m.step()
    torch.cuda.synchronize()
    idx, w, counts = ref.route(host(m.scores), k, score="sigmoid", bias=m.bias.cpu().numpy())
    assert np.array_equal(m.idx.cpu().numpy(), idx) and np.array_equal(m.counts.cpu().numpy(), counts)
    X, bank = unflat(m.X, R, C), m.bank.cpu().numpy()
    Y = ref.forward(oracle, X, bank, idx, w)
    assert near(unflat(m.Y, R, C), Y)
    S = np.array([oracle.sparse_term(np.ascontiguousarray(y.T).reshape(-1)) for y in Y])
    assert np.allclose(m.S.cpu().numpy(), S, rtol=1e-10)
    D = unflat(m.D, R, C)
    Xq = np.transpose(ref.unpack(*ref.pack(m.X.cpu().numpy())).reshape(-1, C, R), (0, 2, 1))
    grad, dF, dw, dX = ref.backward(oracle, D, Xq, bank, idx, w)
    assert near(m.grad.cpu().numpy(), grad, 1e-10) and near(m.dF.cpu().numpy(), dF, 1e-10) and near(m.dw.cpu().numpy(), dw, 1e-10)
    assert near(unflat(m.dX, R, C), dX, 1e-10)
    ds = ref.route_backward(host(m.scores), idx, dw, score="sigmoid")
    # share * (g - mean of g): a difference of parts as large as dw, which agree to 1e-10 of the largest; with one filter
    # per example the difference is zero
    worst = (np.abs(host(m.ds) - ds) - 2.0 ** -24 * np.abs(ds)).max()
    assert worst <= 1e-9 * np.abs(dw).max()


def test_captured_passes(ctx):
    """Two contexts' passes in two graphs, replayed in turn and at once, with eager passes between, against eager results."""
    import torch
    from wavenet_amd import Context
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ms = []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            ms.append(Mixture(Context(0, stream=st.cuda_stream), 70 + 300 * i, 64 if i else 16, 64 if i else 32, 4, 6 + i, 2, i))
    want = []
    for m, st in zip(ms, streams):
        m.step()
        torch.cuda.synchronize()
        want.append(m.results())
    graphs = []
    for m, st in zip(ms, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            m.step()
        graphs.append(g)
    for rep in range(4):
        for m in ms:
            for t in (m.idx, m.counts, m.q):
                t.fill_(-3)
            for t in (m.w, m.Y, m.D, m.S, m.sc, m.grad, m.dF, m.dw, m.dX, m.ds):
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for m, r in zip(ms, want):
            assert all(np.array_equal(a, b) for a, b in zip(m.results(), r)), rep
        ms[0].step()
        torch.cuda.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(ms[0].results(), want[0]))
    del graphs
    for m in ms:
        m.ctx.close()
