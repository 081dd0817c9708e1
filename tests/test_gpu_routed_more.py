"""The routed filter bank beyond the tested sizes' middle: the workgroup kernels in place of the one-wave ones, offsets that
pass 32 bits, other streams, the caller's device."""
import numpy as np
import pytest

import filters as F
import routed_ref as ref
from test_gpu_routed import bank_of, dev, entries, flat, full, host, near, run_backward, run_forward, run_route

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch
    from wavenet_amd import Context
    c = Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    torch.cuda.synchronize()
    c.close()


@pytest.mark.parametrize("R,C,N,k", [(64, 64, 4, 2), (64, 64, 10, 5), (1024, 1, 16, 3), (512, 1, 6, 4), (128, 1, 2, 1)])
def test_workgroup_kernels_agree_with_the_one_wave_kernels(oracle, monkeypatch, R, C, N, k):
    import torch
    from wavenet_amd import Context
    monkeypatch.setenv("WAVENET_HIP_WAVE64", "0")
    c = Context(0, stream=torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(R + N)
    B, F_ = 7, 4
    X, D = rng.standard_normal((B, R, C)), rng.standard_normal((B, R, C))
    bank = bank_of(F_, N, 11)
    idx, w = entries(rng, B, F_, k)
    Y, q, sc = run_forward(c, X, bank, idx, w, keep=True)
    assert near(Y, ref.forward(oracle, X, bank, idx, w))
    rq, rs = ref.pack(np.transpose(X, (0, 2, 1)).reshape(B, -1))
    assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(sc.cpu().numpy(), rs)
    Xq = np.transpose(ref.unpack(rq, rs).reshape(B, C, R), (0, 2, 1))
    for g, r in zip(run_backward(c, D, bank, idx, w, F_, N, q=q, sc=sc), ref.backward(oracle, D, Xq, bank, idx, w)):
        assert near(g, r, 1e-10)
    c.close()


@pytest.mark.parametrize("N", [2, 6, 8, 16, 32])
@pytest.mark.parametrize("R,C", [(32, 32), (16, 16), (64, 16), (1, 512), (1, 1024), (2, 512), (512, 2), (2, 256), (128, 8), (512, 1), (1024, 1)])
@pytest.mark.parametrize("B,k", [(5, 3), (5, 5), (1100, 2)])
def test_one_wave_transforms_in_lds(ctx, oracle, monkeypatch, R, C, N, B, k):
    """Examples of 256 ... 1024 samples whose lines are short, long or single, signals among them where the register kernels
    are off; few and many examples.  Bounds as in the other file: sums of up to 1024 products, errors relative to the largest."""
    import torch
    from wavenet_amd import Context
    c = ctx
    if C == 1:
        monkeypatch.setenv("WAVENET_HIP_WAVE64", "0")
        c = Context(0, stream=torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(R + 5 * C + N)
    F_ = 6
    B = min(B, 1100 if N == 8 else 40)
    X, D = rng.standard_normal((B, R, C)), rng.standard_normal((B, R, C))
    bank = bank_of(F_, N, 17)
    idx, w = entries(rng, B, F_, k)
    assert near(run_forward(c, X, bank, idx, w, keep=False)[0], ref.forward(oracle, X, bank, idx, w))
    for g, r in zip(run_backward(c, D, bank, idx, w, F_, N, X=X), ref.backward(oracle, D, X, bank, idx, w)):
        assert near(g, r, 1e-10)
    if c is not ctx:
        c.close()


@pytest.mark.parametrize("R,C", [(64, 64), (8, 8)])
def test_outputs_over_inputs_are_refused(ctx, R, C):
    import torch
    from wavenet_amd.capi import WavenetError
    B, n, N = 3, R * C, 4
    bank, X = dev(bank_of(1, N, 2)), full((2 * B * n,), 1.5, torch.float64)
    Y, grad, q, sc = (full((B * n,), 9.0, torch.float64), full((B * N,), 9.0, torch.float64), full((8 * B * n,), 3, torch.int8),
                      full((B * -(-n // 64),), 0.5, torch.float32))
    for at in (0, 1, B * n - 1):
        with pytest.raises(WavenetError, match="overlap"):
            ctx.forward_routed(X, B, R, C, bank, None, None, X[at:])
        with pytest.raises(WavenetError, match="overlap"):
            ctx.backprop_routed(Y, B, R, C, bank, None, None, grad, X=X, dX=X[at:])
        with pytest.raises(WavenetError, match="overlap"):
            ctx.backprop_routed(X, B, R, C, bank, None, None, grad, X=Y, dX=X[at:])
    with pytest.raises(WavenetError, match="overlap"):
        ctx.backprop_routed(Y, B, R, C, bank, None, None, grad, q=q, scales=sc, dX=q.view(torch.float64))
    torch.cuda.synchronize()
    assert (X == 1.5).all() and (Y == 9.0).all() and (grad == 9.0).all() and (q == 3).all()
    ctx.forward_routed(X, B, R, C, bank, None, None, X[B * n:])     # one behind the other
    torch.cuda.synchronize()
    assert (X[:B * n] == 1.5).all()


@pytest.mark.parametrize("R,C", [(64, 64), (256, 1), (8, 16)])
@pytest.mark.parametrize("k", [3, 5, 8, 16])
def test_more_filters_than_waves(ctx, oracle, R, C, k):
    """The results of a second round of filters come on top of the first's."""
    rng = np.random.default_rng(k)
    B, F_, N = 600, 20, 8
    X, D = rng.standard_normal((B, R, C)), rng.standard_normal((B, R, C))
    bank = bank_of(F_, N, 5)
    idx, w = entries(rng, B, F_, k)
    some = np.r_[0:6, B - 3:B]
    Y = run_forward(ctx, X, bank, idx, w, keep=False)[0]
    assert near(Y[some], ref.forward(oracle, X[some], bank, idx[some], w[some]))
    grad, dF, dw, dX = run_backward(ctx, D, bank, idx, w, F_, N, X=X)
    rgrad, _, rdw, rdX = ref.backward(oracle, D[some], X[some], bank, idx[some], w[some])
    assert near(grad[some], rgrad, 1e-10) and near(dw[some], rdw, 1e-10) and near(dX[some], rdX, 1e-10)
    want = np.stack([grad[idx == f].sum(axis=0) for f in range(F_)])
    assert near(dF, want, 1e-12)                           # sums of some hundred values in another order


def test_checkpoint_values_in_the_middle(ctx):
    """Values half a scale apart, where the quotient decides: 127 is the block's largest magnitude, so halves are ties."""
    rng = np.random.default_rng(1)
    x = rng.integers(-254, 255, (64, 4096)) / 2.0
    x[:, ::64] = 127.0
    x = x * np.ldexp(1.0, rng.integers(-20, 20, (64, 1)))
    x[5] *= 0.1                                            # no longer ties, but next to them
    x[6] = np.nextafter(x[6], 1e9)
    x[7] = 0.0
    rq, rs = ref.pack(x)
    import torch
    q, sc = full((64, 4096), 0, torch.int8), full((64, 64), 0.0, torch.float32)
    ctx.checkpoint_pack(dev(x), 64, 4096, q, sc)
    torch.cuda.synchronize()
    assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(sc.cpu().numpy(), rs)
    for R, C in ((64, 64), (4096, 1), (2, 2048)):          # the same from the transforms that keep it
        X = np.transpose(x.reshape(64, C, R), (0, 2, 1))
        _, q, sc = run_forward(ctx, X, bank_of(1, 4, 0), None, None, keep=True)
        assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(sc.cpu().numpy(), rs)
    for n in (128, 1024):
        y = x.reshape(-1, n)
        _, q, sc = run_forward(ctx, y[:, :, None], bank_of(1, 4, 0), None, None, keep=True)
        assert np.array_equal(q.cpu().numpy().reshape(64, 4096), rq) and np.array_equal(sc.cpu().numpy().reshape(64, 64), rs)


@pytest.mark.parametrize("R,C", [(64, 64), (512, 1), (16, 16)])
def test_kept_values_that_are_not_finite(ctx, R, C):
    rng = np.random.default_rng(2)
    X = rng.standard_normal((5, R, C))
    X[1, R // 2, C // 2] = np.nan
    X[2, 0, 0] = np.inf
    X[3, R - 1, C - 1] = 1e300
    _, q, sc = run_forward(ctx, X, bank_of(1, 4, 0), None, None, keep=True)
    rq, rs = ref.pack(np.transpose(X, (0, 2, 1)).reshape(5, -1))
    got, want = ref.unpack(q.cpu().numpy(), sc.cpu().numpy()), ref.unpack(rq, rs)
    assert np.array_equal(got, want, equal_nan=True) and np.isnan(got[1:4]).any(axis=1).all()


def test_equal_scores_under_equal_biases_and_many_rows_in_doubt(ctx):
    """bf16 scores repeat; with a bias of zeros, or few different biases, most rows hold values that only the number of the
    filter tells apart, some only 64 bits."""
    import torch
    rng = np.random.default_rng(3)
    for T, F_, k in ((3000, 256, 8), (777, 40, 5), (100, 600, 16)):
        s = dev(rng.standard_normal((T, F_)) * 1.5, torch.bfloat16)
        for bias in (np.zeros(F_), rng.integers(0, 2, F_) * 1e-7, np.full(F_, -0.25), rng.standard_normal(F_) * 1e6):
            for kw in (dict(score="sigmoid"), dict(score="softmax"), dict(score="sigmoid", groups=F_ // 20, groups_kept=2)):
                if F_ % kw.get("groups", 1):
                    continue
                idx, w, counts = run_route(ctx, s, k, bias=dev(bias), **kw)
                ri, rw, rc = ref.route(host(s), k, bias=bias, **kw)
                # values that differ by less than the rounding of 64 bits have no one order: at most a pair in 1e4 rows
                same = (idx == ri).all(axis=1)
                assert same.mean() > 0.999, (T, kw, same.mean())
                assert np.allclose(w[same], rw[same], rtol=2000 * 2.0 ** -53, atol=0)


def test_offsets_beyond_32_bits(ctx, oracle):
    import torch
    # checkpoint: 2.6e9 values
    B, n = 40000, 65536 + 64
    x = torch.zeros(B, n, dtype=torch.bfloat16, device="cuda")
    q, sc = torch.empty(B, n, dtype=torch.int8, device="cuda"), torch.empty(B, n // 64, dtype=torch.float32, device="cuda")
    tail = torch.randn(3, n, device="cuda").to(torch.bfloat16)
    x[-3:] = tail
    q.fill_(5)
    ctx.checkpoint_pack(x, B, n, q, sc)
    torch.cuda.synchronize()
    rq, rs = ref.pack(host(tail))
    assert np.array_equal(q[-3:].cpu().numpy(), rq) and np.array_equal(sc[-3:].cpu().numpy(), rs) and not q[:-3].any() and not sc[:-3].any()
    x.fill_(1.0)
    ctx.checkpoint_unpack(q, sc, B, n, x)
    torch.cuda.synchronize()
    assert np.array_equal(host(x[-3:]), host(torch.from_numpy(ref.unpack(rq, rs)).to(torch.bfloat16))) and not x[:-3].any()
    del x, q, sc
    # router: 4.8e9 scores
    T, F_ = 9_400_000, 512
    s = torch.zeros(T, F_, dtype=torch.float16, device="cuda")
    last = torch.randn(2, F_, device="cuda").to(torch.float16)
    s[-2:] = last
    idx, w = torch.empty(T, 2, dtype=torch.int32, device="cuda"), torch.empty(T, 2, dtype=torch.float64, device="cuda")
    counts = torch.empty(F_, dtype=torch.int32, device="cuda")
    ctx.route(s, T, F_, idx, w, k=2, counts=counts)
    torch.cuda.synchronize()
    ri, rw, _ = ref.route(host(last), 2)
    assert np.array_equal(idx[-2:].cpu().numpy(), ri) and np.allclose(w[-2:].cpu().numpy(), rw, rtol=1e-12)
    assert (idx[:-2] == torch.tensor([0, 1], dtype=torch.int32, device="cuda")).all() and int(counts.sum()) == 2 * T
    ctx.route_backward(s, T, F_, idx, w, s, k=2, renormalise=False)
    torch.cuda.synchronize()
    want = ref.route_backward(host(last), ri, rw, renormalise=False)
    assert (np.abs(host(s[-2:]) - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()
    del s, idx, w
    # transforms: 5.2e9 bytes of examples
    B, R, C = 160000, 64, 64
    rng = np.random.default_rng(4)
    X = torch.zeros(B, R * C, dtype=torch.float64, device="cuda")
    Y = torch.empty_like(X)
    end = rng.standard_normal((2, R, C))
    X[-2:] = flat(end)
    bank = bank_of(2, 4, 0)
    idx = torch.ones(B, 1, dtype=torch.int32, device="cuda")
    w = torch.ones(B, 1, dtype=torch.float64, device="cuda")
    ctx.forward_routed(X, B, R, C, dev(bank), idx, w, Y)
    torch.cuda.synchronize()
    one = np.ones((2, 1), dtype=np.int32)
    got = np.transpose(Y[-2:].cpu().numpy().reshape(2, C, R), (0, 2, 1))
    assert near(got, ref.forward(oracle, end, bank, one, np.ones((2, 1)))) and not Y[:-2].any()


def test_another_stream_and_the_callers_device(oracle):
    """Work goes to the context's stream in order with what the caller queued there, and the current device stays."""
    import torch
    from wavenet_amd import Context
    st = torch.cuda.Stream()
    c = Context(0, stream=st.cuda_stream)
    rng = np.random.default_rng(6)
    B, R, C = 200, 64, 64
    X = rng.standard_normal((B, R, C))
    bank = bank_of(3, 4, 0)
    idx, w = entries(rng, B, 3, 2)
    dX, dbank, didx, dw = flat(X), dev(bank), dev(idx), dev(w)
    torch.cuda.synchronize()
    before = torch.cuda.current_device()
    with torch.cuda.stream(st):
        twice = dX * 2.0
        Y = torch.empty_like(twice)
        c.forward_routed(twice, B, R, C, dbank, didx, dw, Y)
        Z = Y * 0.5
    st.synchronize()
    assert torch.cuda.current_device() == before
    got = np.transpose(Z.cpu().numpy().reshape(B, C, R), (0, 2, 1))
    some = np.r_[0:8]
    assert near(got[some], ref.forward(oracle, X[some], bank, idx[some], w[some]))
    c.close()


@pytest.mark.parametrize("T,F_,k", [(5, 1024, 16), (700, 96, 3)])
@pytest.mark.parametrize("dtype", ["float64", "float32", "bfloat16"])
def test_all_groups_kept_is_no_groups(ctx, T, F_, k, dtype):
    """Any number of groups, one per filter too, if all of them are kept."""
    import torch
    rng = np.random.default_rng(F_)
    s = dev(rng.standard_normal((T, F_))).to(getattr(torch, dtype))
    bias = dev(rng.standard_normal(F_) * 0.1)
    for b in (None, bias):
        want = run_route(ctx, s, k, bias=b)
        for groups in (2, F_ // 3 if F_ % 3 == 0 else F_ // 4, F_):
            got = run_route(ctx, s, k, bias=b, groups=groups, groups_kept=groups)
            assert all(np.array_equal(g, w) for g, w in zip(got, want))


def test_contexts_of_different_sizes(ctx):
    """Two contexts on one GPU whose launches of the same kernels need different amounts of LDS, in turn."""
    import torch
    from wavenet_amd import Context
    other = Context(0, stream=torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(8)
    big, small = dev(rng.standard_normal((40, 1024))), dev(rng.standard_normal((40, 640)))
    bank = dev(bank_of(2, 4, 3))
    X = [dev(rng.standard_normal((4, 64 * 64))) for _ in range(2)]
    D = dev(rng.standard_normal((4, 64 * 64)))
    first = None
    for turn in range(3):
        out = [run_route(c, s, 5, groups=16, groups_kept=4) for c, s in ((ctx, big), (other, small))]
        for c, k in ((ctx, 4), (other, 2)):
            idx = full((4, k), 1, torch.int32)
            Y, grad, dX = full((4, 4096), 0.0, torch.float64), full((4, k, 4), 0.0, torch.float64), full((4, 4096), 0.0, torch.float64)
            c.forward_routed(X[0], 4, 64, 64, bank, idx, None, Y)
            c.backprop_routed(D, 4, 64, 64, bank, idx, None, grad, X=X[0], dX=dX)
            torch.cuda.synchronize()
            out.append([t.cpu().numpy() for t in (Y, grad, dX)])
        if first is None:
            first = out
        assert all(np.array_equal(a, b) for x, y in zip(out, first) for a, b in zip(x, y))
    other.close()
