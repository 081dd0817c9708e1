"""The routed filter bank where values say that there is no answer, lie next to each other, or share memory."""
import numpy as np
import pytest

import routed_ref as ref
from test_gpu_routed import bank_of, dev, flat, full, host, near, run_backward, run_forward, run_route, torch_type, unflat

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


@pytest.mark.parametrize("dtype", ["f64", "f32", "f16", "bf16"])
def test_route_tells_equal_shares_apart_by_their_scores(ctx, dtype):
    """Without a bias: sigmoids that are 1 and shares of a softmax that are 0 in 64 bits.  With one the shares are what counts."""
    s = np.array([[40.0, 50.0, 44.0, 60.0, 48.0, 39.0, -1.0, 56.0], [-900.0, -800.0, 0.0, -850.0, -1000.0, -810.0, -950.0, -1100.0]])
    v = dev(s, torch_type(dtype))
    for score in ("sigmoid", "softmax"):
        idx, _, _ = run_route(ctx, v, 4, score=score)
        assert np.array_equal(idx, [[3, 7, 1, 4], [2, 1, 5, 3]])
    ones = dev(np.ones(8))
    assert np.array_equal(run_route(ctx, v, 4, score="sigmoid", bias=ones)[0][0], [0, 1, 2, 3])
    assert np.array_equal(run_route(ctx, v, 4, bias=ones)[0][1], [2, 0, 1, 3])


@pytest.mark.parametrize("F_,groups,kept,k", [(129, 43, 5, 9), (65, 65 // 5, 4, 6), (513, 57, 3, 16), (576, 64, 9, 16), (1000, 50, 7, 16), (33, 33, 8, 5)])
def test_route_groups_that_end_inside_a_lane(ctx, F_, groups, kept, k):
    """Lanes past the last filter, whose numbers would make groups past the last."""
    rng = np.random.default_rng(F_)
    s = rng.standard_normal((50, F_))
    bias = rng.standard_normal(F_) * 0.05
    for b in (None, bias):
        for kw in (dict(score="sigmoid"), dict(renormalise=False)):
            got = run_route(ctx, dev(s), k, groups=groups, groups_kept=kept, bias=None if b is None else dev(b), **kw)
            want = ref.route(s, k, groups=groups, groups_kept=kept, bias=b, **kw)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[2], want[2])
            assert np.allclose(got[1], want[1], rtol=2000 * 2.0 ** -53, atol=0)


def test_route_chosen_again_in_groups_and_counted(ctx):
    """Rows that the 32-bit values leave in doubt, most of a batch: the counts are those of the indices that left, and a row that
    differs from the reference holds values that 64 bits do not tell apart.  p is within 2000 * 2^-53 of itself (as the weights
    are), p + bias rounds by half a unit of 2^-52 |c| on either side, a group's score is the sum of two."""
    import torch
    rng = np.random.default_rng(9)
    for T, F_, k, groups in ((600, 256, 8, 16), (777, 40, 5, 8), (100, 600, 16, 30)):
        wide = rng.standard_normal((T, F_))
        for scores, dtype in ((wide * 1.5, torch.bfloat16), (wide * 40.0, torch.bfloat16), (wide * 40.0, torch.float32), (wide * 40.0, torch.float64)):
            s = dev(scores).to(dtype)
            for bias in (None, np.zeros(F_), rng.integers(0, 2, F_) * 1e-7, rng.standard_normal(F_) * 1e6):
                for kw in (dict(score="sigmoid", groups=groups, groups_kept=3), dict(groups=groups, groups_kept=2)):
                    idx, w, counts = run_route(ctx, s, k, bias=None if bias is None else dev(bias), **kw)
                    assert np.array_equal(counts, np.bincount(idx[idx >= 0], minlength=F_))
                    ri, rw, _ = ref.route(host(s), k, bias=bias, **kw)
                    same = (idx == ri).all(axis=1)
                    assert np.allclose(w[same], rw[same], rtol=2000 * 2.0 ** -53, atol=0)
                    if same.all():
                        continue
                    p = ref.shares(host(s), kw.get("score", "softmax"))
                    c = p if bias is None else p + bias
                    bound = 2 * (2 * 2000 * 2.0 ** -53 + 4 * 2.0 ** -53 * np.abs(c).max())
                    best = np.sort(c.reshape(T, groups, -1), axis=2)[:, :, -2:].sum(axis=2)
                    order = np.sort(best, axis=1)[:, ::-1]
                    kept = kw["groups_kept"]
                    for t in np.flatnonzero(~same):
                        assert (idx[t] >= 0).all() and len(set(idx[t])) == k
                        near_groups = order[t, kept - 1] - order[t, kept] <= bound
                        # (without a bias filters of a group are told apart by their scores, which are exact)
                        near_values = bias is not None and (np.abs(c[t, idx[t]] - c[t, ri[t]]) <= bound).all()
                        assert near_groups or near_values, (T, kw, t)


# ---- refusals -------------------------------------------------------------------------------------------------------

def test_a_refused_backward_pass_has_written_nothing(ctx):
    import torch
    from wavenet_amd import capi
    B, n, N = 3, 64, 4
    D, X, bank = full((B, n), 1.0, torch.float64), full((B, n), 2.0, torch.float64), dev(bank_of(2, N, 0))
    grad, dw, dX = full((B, 1, N), 9.0, torch.float64), full((B, 1), 9.0, torch.float64), full((B, n), 9.0, torch.float64)
    dF = full((2 * N + 1,), 9.0, torch.float64)
    with pytest.raises(capi.WavenetError) as err:
        ctx.backprop_routed(D, B, 8, 8, bank, None, None, grad, X=X, dw=dw, dX=dX, dfilters=dF.data_ptr() + 4)
    assert err.value.status == capi.WN_ERR_ARG
    torch.cuda.synchronize()
    assert all((t == 9.0).all() for t in (grad, dw, dX, dF))


def test_layouts_other_than_the_strides_are_refused(ctx):
    """A tensor whose own strides are not the ones passed would be read as other values than the caller's."""
    import torch
    rng = np.random.default_rng(0)
    T, F_, k = 12, 8, 2
    s = rng.standard_normal((T, F_))
    idx, w = full((T, k), 0, torch.int32), full((T, k), 0.0, torch.float64)
    turned, gaps = dev(s.T.copy()).t(), dev(np.repeat(s, 2, axis=1))[:, ::2]
    ri, rw, _ = ref.route(s, k)
    for v in (turned, gaps):
        with pytest.raises(ValueError, match="strides"):
            ctx.route(v, T, F_, idx, w, k=k)
        with pytest.raises(ValueError, match="strides"):
            ctx.route_backward(dev(s), T, F_, idx, w, v, k=k)
        with pytest.raises(ValueError, match="strides"):
            ctx.route_backward(v, T, F_, idx, w, dev(s), k=k)
        with pytest.raises(ValueError, match="strides"):
            ctx.checkpoint_pack(v, T, F_, full((T, F_), 0, torch.int8), full((T, 1), 0.0, torch.float32))
        with pytest.raises(ValueError, match="strides"):
            ctx.checkpoint_unpack(full((T, F_), 0, torch.int8), full((T, 1), 0.0, torch.float32), T, F_, v)
        gi, gw, _ = run_route(ctx, v, k)                            # with its strides
        assert np.array_equal(gi, ri) and np.allclose(gw, rw, rtol=2000 * 2.0 ** -53, atol=0)
    with pytest.raises(ValueError, match="strides"):
        ctx.route(turned, T, F_, idx, w, k=k, row_stride=1, col_stride=F_)      # (a column is T scores long)


def test_tables_of_another_width_are_refused(ctx):
    """Indices, weights and filters of two dimensions are rows of k and of N: any other width would be read out of step."""
    import torch
    B, n, N = 6, 64, 4
    X, Y, bank = full((B, n), 1.0, torch.float64), full((B, n), 9.0, torch.float64), dev(bank_of(3, N, 0))
    two, three = full((B, 2), 0, torch.int32), full((B, 3), 0, torch.int32)
    w2, w3 = full((B, 2), 9.0, torch.float64), full((B, 3), 9.0, torch.float64)
    grad = full((B, 2, N), 9.0, torch.float64)
    s = full((B, 8), 0.0, torch.float64)
    with pytest.raises(ValueError, match="wide"):
        ctx.forward_routed(X, B, 8, 8, bank, two, w3, Y)
    with pytest.raises(ValueError, match="wide"):
        ctx.forward_routed(X, B, 8, 8, bank, three, w3, Y, k=2)
    with pytest.raises(ValueError, match="wide"):
        ctx.forward_routed(X, B, 8, 8, bank, two, w2, Y, N=2)
    for kw in (dict(dw=w3), dict(grad=full((B, 3, N), 9.0, torch.float64)), dict(grad=full((B, 2, N + 1), 9.0, torch.float64)),
               dict(dfilters=full((3, N + 2), 9.0, torch.float64))):
        with pytest.raises(ValueError, match="wide"):
            ctx.backprop_routed(Y, B, 8, 8, bank, two, w2, **{"grad": grad, "X": X, **kw})
    with pytest.raises(ValueError, match="wide"):
        ctx.route(s, B, 8, three, w2, k=2)
    with pytest.raises(ValueError, match="wide"):
        ctx.route(s, B, 8, two, w3, k=2)
    with pytest.raises(ValueError, match="wide"):
        ctx.route_backward(s, B, 8, two, w3, s.clone(), k=2)
    torch.cuda.synchronize()
    assert (Y == 9.0).all() and (grad == 9.0).all() and (w2 == 9.0).all() and not two.any()


@pytest.mark.parametrize("from_checkpoint", [False, True])
def test_every_output_over_every_other_argument_is_refused(ctx, from_checkpoint):
    """By a byte at either end; what lies side by side is taken, and a refused call has written nothing."""
    import torch
    from wavenet_amd import capi
    B, R, C, N, F_, k = 3, 8, 16, 4, 5, 2
    n, nb = R * C, R * C // 64
    nbytes = dict(X=8 * B * n, filters=8 * F_ * N, idx=4 * B * k, w=8 * B * k, Y=8 * B * n, q=B * n, scales=4 * B * nb, Delta=8 * B * n,
                  grad=8 * B * k * N, dfilters=8 * F_ * N, dw=8 * B * k, dX=8 * B * n)
    align = dict(idx=4, scales=4, q=1)
    room = 64 * (sum(nbytes.values()) // 64 + 2 * len(nbytes))
    # the arguments of one call after the other, without a gap but for alignment
    arena = torch.zeros(3 * room, dtype=torch.uint8, device="cuda")
    base, at, end = arena.data_ptr(), {}, arena.data_ptr() + room
    for name, size in sorted(nbytes.items(), key=lambda item: -align.get(item[0], 8)):
        at[name] = end
        end += size
    used = end - base

    def forward(a):
        ctx.forward_routed(a["X"], B, R, C, a["filters"], a["idx"], a["w"], a["Y"], k=k, F=F_, N=N, q=a["q"], scales=a["scales"])

    def backward(a):
        src = dict(q=a["q"], scales=a["scales"]) if from_checkpoint else dict(X=a["X"])
        ctx.backprop_routed(a["Delta"], B, R, C, a["filters"], a["idx"], a["w"], a["grad"], dfilters=a["dfilters"], dw=a["dw"], dX=a["dX"], k=k,
                            F=F_, N=N, **src)

    back_in = ["Delta", "filters", "idx", "w"] + (["q", "scales"] if from_checkpoint else ["X"])
    tried = 0
    for call, outputs, inputs in ((forward, ["Y", "q", "scales"], ["X", "filters", "idx", "w"]), (backward, ["grad", "dfilters", "dw", "dX"], back_in)):
        call(at)
        torch.cuda.synchronize()
        before = arena.clone()
        for o in outputs:
            for other in [x for x in inputs + outputs if x != o]:
                step = align.get(o, 8)
                first = at[other] - nbytes[o] + step                    # the last element of o on the first of the other
                last = at[other] + nbytes[other] - step                 # and the other way round
                for address in (first + -(first - base) % step, last - (last - base) % step, at[other] + -(at[other] - base) % step):
                    with pytest.raises(capi.WavenetError, match="overlaps") as err:
                        call({**at, o: address})
                    assert err.value.status == capi.WN_ERR_ARG
                    tried += 1
        torch.cuda.synchronize()
        assert torch.equal(arena, before)
    assert tried >= 3 * 3 * 6 and used <= arena.numel()


def test_router_and_checkpoint_outputs_over_inputs_are_refused(ctx):
    import torch
    from wavenet_amd import capi
    rng = np.random.default_rng(3)
    T, F_, k, gap = 4, 8, 2, 40
    arena = dev(np.zeros(4 * T * (F_ + gap)))
    base, row = arena.data_ptr() + 8 * T * (F_ + gap), 8 * (F_ + gap)
    view = arena[T * (F_ + gap):2 * T * (F_ + gap)].view(T, F_ + gap)[:, :F_]
    s = rng.standard_normal((T, F_))
    view.copy_(dev(s))
    idx, w, bias, counts = full((T, k), 0, torch.int32), full((T, k), 0.0, torch.float64), dev(np.zeros(F_)), full((F_,), 0, torch.int32)
    spare = full((T, F_), 0.0, torch.float64)
    torch.cuda.synchronize()

    def refused(fn, *a, **kw):
        before = arena.clone()
        with pytest.raises(capi.WavenetError, match="overlap") as err:
            fn(*a, **kw)
        assert err.value.status == capi.WN_ERR_ARG
        torch.cuda.synchronize()
        assert torch.equal(arena, before)

    by_rows, by_filters = dict(row_stride=F_ + gap, col_stride=1), dict(row_stride=1, col_stride=F_ + gap)
    for strides, T_, n in ((by_rows, T, F_), (by_filters, F_, T)):
        for at in (base, base + row + 8 * (F_ - 1), base + 3 * row, base - 8 * T_ * k + 8, base + row - 8):
            refused(ctx.route, base, T_, n, idx.data_ptr() if T_ == T else spare.data_ptr(), at, k=k, **strides)
        refused(ctx.route, base, T_, n, base + 2 * row + 8, w.data_ptr() if T_ == T else spare.data_ptr(), k=k, **strides)
        refused(ctx.route, base, T_, n, spare.data_ptr(), spare.data_ptr() + 128, k=k, counts=base, **strides)
    refused(ctx.route, base, T, F_, idx, bias.data_ptr() - 8, k=k, bias=bias, **by_rows)
    refused(ctx.route, base, T, F_, w.data_ptr(), w.data_ptr() + 8, k=k, **by_rows)
    refused(ctx.route, base, T, F_, idx, w, k=k, counts=idx.data_ptr() + 4 * T * k - 4, **by_rows)
    # between the rows of the scores there is room
    between = base + row + 8 * F_
    ctx.route(base, T, F_, idx, between, k=k, counts=counts, **by_rows)
    torch.cuda.synchronize()
    ri, rw, rc = ref.route(s, k)
    got = arena[T * (F_ + gap) + F_ + gap + F_:][:T * k].cpu().numpy().reshape(T, k)
    assert np.array_equal(idx.cpu().numpy(), ri) and np.allclose(got, rw, rtol=2000 * 2.0 ** -53, atol=0) and np.array_equal(counts.cpu().numpy(), rc)

    # gradients: on their own scores, beside them, or between the rows; not on other scores, indices or weights
    dw = dev(rng.standard_normal((T, k)))
    want = ref.route_backward(s, ri, dw.cpu().numpy())
    for at in (8, -8, row, -row, 3 * row, row + 16, 8 * (F_ - 1), -2 * row + 8 * (F_ - 1)):
        refused(ctx.route_backward, base, T, F_, idx, dw, base + at, k=k, **by_rows)
    refused(ctx.route_backward, base, T, F_, idx, base + row + 8 * (F_ + 2), base + 16, k=k, **by_rows)
    refused(ctx.route_backward, base, T, F_, idx, base + row + 8 * (F_ + 2), base + 8 * (F_ + 2), k=k, **by_rows)
    refused(ctx.route_backward, base, T, F_, base + 3 * row + 8 * (F_ + 1), dw, base + 8 * F_, k=k, **by_rows)
    for at in (8 * F_, -8 * F_, 4 * row, -4 * row):
        out = base + at
        ctx.route_backward(base, T, F_, idx, dw, out, k=k, **by_rows)
        torch.cuda.synchronize()
        first = (out - arena.data_ptr()) // 8
        got = arena.as_strided((T, F_), (F_ + gap, 1), first).cpu().numpy()
        assert (np.abs(got - want) <= 1e-11 * max(1.0, np.abs(want).max())).all() and np.array_equal(view.cpu().numpy(), s)

    # checkpoints
    q, sc = full((T, F_), 0, torch.int8), full((T,), 0.0, torch.float32)
    for a in ((base, sc.data_ptr()), (base + 2 * row + 8 * F_ - 1, sc.data_ptr()), (q.data_ptr(), base + row), (q.data_ptr(), base - 12),
              (q.data_ptr(), q.data_ptr() + T * F_ - 4)):
        refused(ctx.checkpoint_pack, base, T, F_, *a, row_stride=F_ + gap)
    for a in ((base, sc.data_ptr()), (q.data_ptr(), base + row)):
        refused(ctx.checkpoint_unpack, *a, T, F_, base, row_stride=F_ + gap)
    ctx.checkpoint_pack(base, T, F_, base + 8 * F_, base + 8 * F_ + T * F_, row_stride=F_ + gap)      # between two rows
    ctx.checkpoint_unpack(base + 8 * F_, base + 8 * F_ + T * F_, T, F_, spare)
    torch.cuda.synchronize()
    assert np.array_equal(spare.cpu().numpy(), ref.unpack(*ref.pack(s))) and np.array_equal(view.cpu().numpy(), s)


# ---- together -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("R,C,N,k", [(64, 64, 4, 2), (16, 32, 6, 3), (512, 1, 8, 2)])
def test_examples_routed_by_their_costs_under_a_grid_of_filters(ctx, oracle, R, C, N, k):
    """From wn_sparse_cost_grid's costs, filter by filter, to the gradients of the filters that suit an example best."""
    import torch
    rng = np.random.default_rng(R + k)
    B, F_, n, cold = 21, 9, R * C, 0.05
    X = rng.random((B, R, C)) ** 4
    bank = bank_of(F_, N, 60)
    S = full((F_, B), -1.0, torch.float64)
    ctx.sparse_cost_grid(flat(X), B, R, C, bank, S)
    idx, w, counts = full((B, k), -7, torch.int32), full((B, k), 7.0, torch.float64), full((F_,), -7, torch.int32)
    how = dict(k=k, score_scale=-1.0 / cold)
    ctx.route(S, B, F_, idx, w, row_stride=1, col_stride=B, counts=counts, **how)
    torch.cuda.synchronize()
    costs = S.cpu().numpy().T
    want = np.array([[oracle.sparse_term(np.ascontiguousarray(oracle.band_forward_2d(a, x)[3].T).reshape(-1)) for a in bank] for x in X])
    assert np.allclose(costs, want, rtol=1e-10)
    ri, rw, rc = ref.route(costs, k, score_scale=-1.0 / cold)
    assert np.array_equal(idx.cpu().numpy(), ri) and np.array_equal(counts.cpu().numpy(), rc)
    assert np.allclose(w.cpu().numpy(), rw, rtol=2000 * 2.0 ** -53, atol=0)
    assert np.array_equal(ri[:, 0], costs.argmin(axis=1))               # the sparsest comes first
    Y, q, sc = run_forward(ctx, X, bank, ri, rw, keep=True)
    assert near(Y, ref.forward(oracle, X, bank, ri, rw))
    D, T = full((B, n), 7.0, torch.float64), full((B,), 7.0, torch.float64)
    ctx.sparse_term_deriv(flat(Y), B, n, D, T)
    torch.cuda.synchronize()
    got = run_backward(ctx, unflat(D, R, C), bank, ri, rw, F_, N, q=q, sc=sc)
    Xq = np.transpose(ref.unpack(*ref.pack(np.transpose(X, (0, 2, 1)).reshape(B, n))).reshape(B, C, R), (0, 2, 1))
    for g, r in zip(got, ref.backward(oracle, unflat(D, R, C), Xq, bank, ri, rw)):
        assert near(g, r, 1e-10)
    assert not got[1][rc == 0].any()
    ds = full((F_, B), 7.0, torch.float64)
    ctx.route_backward(S, B, F_, dev(ri), dev(got[2]), ds, row_stride=1, col_stride=B, **how)
    torch.cuda.synchronize()
    want = ref.route_backward(costs, ri, got[2], score_scale=-1.0 / cold)
    assert (np.abs(ds.cpu().numpy().T - want) <= 1e-10 * max(1.0, np.abs(got[2]).max()) / cold).all()
