"""What is measured of the routed filter bank: the router, its backward pass, 8-bit checkpoints of activations, the
transforms of examples under the filters they were routed to, and their backward pass.

Examples are fp64 and column-major (sample (r, c) at r + c*R), a batch is contiguous; a filter is a row of N low-pass
taps.  `run` computes the plain form from elementary torch operations, or (own = True) calls the framework.  The plain
form works in 64 bits throughout: the transforms' arrays are fp64, and the router compares values next to a border.
"""
import math

import torch

own = False

_DTYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
_BLOCK = 64  # values that share one scale in a checkpoint


# ---- cases ----------------------------------------------------------------------------------------------------

def _route(name, kind, T, F, k, dtype, score="softmax", bias=False, groups=1, kept=1, renorm=True, scale=1.0,
           score_scale=1.0, by_filter=False):
    case = dict(kind=kind, T=T, F=F, k=k, dtype=dtype, score=score, bias=bias, groups=groups, kept=kept, renorm=renorm,
                scale=scale, score_scale=score_scale, by_filter=by_filter)
    return dict(name=name, **case) if name else case


def _bank(name, kind, B, R, C, N, F, k):
    case = dict(kind=kind, B=B, R=R, C=C, N=N, F=F, k=k)
    return dict(name=name, **case) if name else case


def _checkpoint(name, B, n, dtype):
    case = dict(kind="checkpoint", B=B, n=n, dtype=dtype)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one example that arrives by itself, eight filters: only latency counts
        _route("route-1x8", "route", 1, 8, 2, "f32"),
        # the headline batch routed by its sparsity costs under a grid of filters: fp64, filter-major, lower is better
        _route("route-costs-4096x256", "route", 4096, 256, 2, "f64", score_scale=-8.0, by_filter=True),
        # the largest: a long stream of half-precision scores of a learned router, balance bias and groups
        _route("route-groups-65536x256", "route", 65536, 256, 8, "bf16", score="sigmoid", bias=True, groups=8, kept=4,
               scale=2.5),
        # gradient of the headline batch's scores, renormalised pair of filters
        _route("route-grad-4096x64", "route_grad", 4096, 64, 2, "f32"),
        # gradient of a long stream of scores through the full softmax
        _route("route-grad-65536x256", "route_grad", 65536, 256, 8, "bf16", renorm=False),
        # a few activations of odd length from a program that works in 32 bits
        _checkpoint("checkpoint-37x777", 37, 777, "f32"),
        # the headline batch's input as a checkpoint and back
        _checkpoint("checkpoint-4096x4096", 4096, 4096, "f64"),
        # one image by itself under its two filters (applying a trained bank)
        _bank("forward-1x64x64", "forward", 1, 64, 64, 4, 8, 2),
        # the headline batch under two of sixteen filters
        _bank("forward-4096x64x64", "forward", 4096, 64, 64, 4, 16, 2),
        # training pass over the headline batch: forward that keeps a checkpoint, backward that reads it
        _bank("train-4096x64x64", "train", 4096, 64, 64, 4, 16, 2),
        # training pass over small odd-shaped images in an odd batch, four filters each
        _bank("train-1000x16x32", "train", 1000, 16, 32, 8, 32, 4),
        # backward pass of the signals of the 1D workload, from a checkpoint kept earlier
        _bank("backward-777x1024x1", "backward", 777, 1024, 1, 16, 64, 2),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["route", "route_grad", "checkpoint", "forward", "train", "backward"])
    if kind in ("route", "route_grad"):
        F = _spread(rng, 2, 512)
        T = _spread(rng, 1, min(65536, (65536 * 256) // F))
        score = rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16) if F % g == 0])
        kept = rng.randint(1, groups)
        return _route(None, kind, T, F, rng.randint(1, min(8, F)), rng.choice(sorted(_DTYPES)), score, rng.random() < 0.5,
                      groups, kept, rng.random() < 0.6, rng.choice([1.0, 2.5]), rng.choice([1.0, 0.5, -8.0]),
                      rng.random() < 0.3)
    if kind == "checkpoint":
        n = _spread(rng, 1, 16384)
        return _checkpoint(None, _spread(rng, 1, min(16384, (4096 * 4096) // n)), n, rng.choice(sorted(_DTYPES)))
    R, C = rng.choice([(64, 64), (1024, 1), (512, 1), (256, 1), (4096, 1), (16, 32), (32, 8), (2, 1024), (1, 64), (32, 64),
                       (128, 1), (8, 8), (2, 2), (64, 1)])
    N = rng.choice([2, 4, 6, 8, 10, 16])
    k = rng.randint(1, 4)
    # no more work than the largest listed pass: samples times taps times filters an example
    room = (4096 * 4096 * 4 * 2) // (R * C * N * k)
    return _bank(None, kind, _spread(rng, 1, max(1, min(8192, room))), R, C, N, _spread(rng, k, 64), k)


# ---- inputs ---------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _filters(F, N, g):
    """F filters of N taps near the unit-norm sphere on which filters are initialised and stay close to."""
    a = torch.randn(F, N, dtype=torch.float64, device="cuda", generator=g)
    return a / a.norm(dim=1, keepdim=True)


def _pick(B, F, k, g):
    """k different filters of F for each example, and weights that sum to one."""
    idx = torch.rand(B, F, device="cuda", generator=g).topk(k, dim=1).indices.to(torch.int32)
    w = torch.rand(B, k, dtype=torch.float64, device="cuda", generator=g) + 0.1
    return idx.contiguous(), w / w.sum(dim=1, keepdim=True)


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    s = dict(case=dict(case))
    f64 = dict(dtype=torch.float64, device="cuda")
    if own:
        from wavenet_amd import Context
        s["ctx"] = Context(torch.cuda.current_device(), stream=torch.cuda.current_stream().cuda_stream)
    if kind in ("route", "route_grad"):
        T, F, k = case["T"], case["F"], case["k"]
        if case["score_scale"] < 0:   # sparsity costs: between 0 and 1
            v = torch.rand(T, F, generator=g, **f64)
        else:
            v = torch.randn(T, F, generator=g, **f64) * 1.5
        v = v.to(_DTYPES[case["dtype"]])
        v = v.t().contiguous().t() if case["by_filter"] else v.contiguous()
        s["scores"] = v
        s["bias"] = torch.randn(F, generator=g, **f64) * 0.05 if case["bias"] else None
        if kind == "route":
            s["idx"] = torch.empty(T, k, dtype=torch.int32, device="cuda")
            s["w"] = torch.empty(T, k, **f64)
            s["counts"] = torch.empty(F, dtype=torch.int32, device="cuda")
        else:
            s["idx"] = _plain_route(v, s["bias"], case)[0]
            s["dw"] = torch.randn(T, k, generator=g, **f64)
            s["dscores"] = torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device="cuda")
        return s
    if kind == "checkpoint":
        B, n = case["B"], case["n"]
        # activations: mostly small, a few large
        v = torch.randn(B, n, generator=g, **f64) * torch.exp(torch.randn(B, n, generator=g, **f64))
        s["X"] = v.to(_DTYPES[case["dtype"]])
        s["q"] = torch.empty(B, n, dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty(B, -(-n // _BLOCK), dtype=torch.float32, device="cuda")
        s["out"] = torch.empty_like(s["X"])
        return s
    B, n, N, F, k = case["B"], case["R"] * case["C"], case["N"], case["F"], case["k"]
    s["filters"] = _filters(F, N, g)
    s["idx"], s["w"] = _pick(B, F, k, g)
    X = torch.rand(B, n, generator=g, **f64)
    nb = -(-n // _BLOCK)
    if kind == "backward":
        s["q"], s["scales"] = _plain_pack(X)
    else:
        s["X"] = X
        s["Y"] = torch.empty(B, n, **f64)
    if kind == "train":
        s["q"] = torch.empty(B, n, dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty(B, nb, dtype=torch.float32, device="cuda")
    if kind != "forward":
        s["D"] = torch.randn(B, n, generator=g, **f64)
        s["grad"] = torch.empty(B, k, N, **f64)
        s["dfilters"] = torch.empty(F, N, **f64)
        s["dw"] = torch.empty(B, k, **f64)
        s["dX"] = torch.empty(B, n, **f64)
    return s


# ---- plain form -----------------------------------------------------------------------------------------------

def _top(c, k):
    """k largest of every row, descending, ties to the lowest index; closed entries are -inf."""
    order = torch.argsort(c, dim=1, descending=True, stable=True)[:, :k]
    return order, torch.gather(c, 1, order)


def _plain_scores(scores, case):
    s = scores.to(torch.float64) * case["score_scale"]
    if case["score"] == "softmax":
        e = torch.exp(s - s.amax(dim=1, keepdim=True))
        return s, e / e.sum(dim=1, keepdim=True)
    return s, 1.0 / (1.0 + torch.exp(-s))


def _plain_route(scores, bias, case):
    T, F, k, G, kept = case["T"], case["F"], case["k"], case["groups"], case["kept"]
    s, p = _plain_scores(scores, case)
    c = s if bias is None else p + bias
    if kept < G:
        cg = (p if bias is None else c).reshape(T, G, F // G)
        best = torch.sort(cg, dim=2, descending=True).values[:, :, :2].sum(dim=2)
        keep = torch.zeros(T, G, dtype=torch.bool, device=scores.device)
        keep.scatter_(1, _top(best, kept)[0], True)
        c = torch.where(keep.repeat_interleave(F // G, dim=1), c, torch.full_like(c, -math.inf))
    order, got = _top(c, k)
    if order.shape[1] < k:
        raise ValueError("k exceeds the number of filters")
    w = torch.gather(p, 1, order)
    open_ = got > -math.inf
    w = torch.where(open_, w, torch.zeros_like(w))
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    idx = torch.where(open_, order, torch.full_like(order, -1)).to(torch.int32)
    counts = torch.zeros(F + 1, dtype=torch.int32, device=scores.device)
    counts.index_add_(0, torch.where(open_, order, torch.full_like(order, F)).reshape(-1),
                      torch.ones(T * k, dtype=torch.int32, device=scores.device))
    return idx, w * case["scale"], counts[:F]


def _plain_route_grad(scores, idx, dw, case):
    _, p = _plain_scores(scores, case)
    at = idx.clamp(min=0).to(torch.int64)
    live = (idx >= 0).to(torch.float64)
    pj = torch.gather(p, 1, at) * live
    g = dw * live * case["scale"]
    if case["renorm"]:
        u = pj / pj.sum(dim=1, keepdim=True)
        d = u * (g - (u * g).sum(dim=1, keepdim=True))
        if case["score"] == "sigmoid":
            d = d * (1.0 - pj)
        ds = torch.zeros_like(p).scatter_add_(1, at, d)
    elif case["score"] == "sigmoid":
        ds = torch.zeros_like(p).scatter_add_(1, at, g * pj * (1.0 - pj))
    else:
        ds = p * (torch.zeros_like(p).scatter_add_(1, at, g) - (g * pj).sum(dim=1, keepdim=True))
    return (ds * case["score_scale"]).to(scores.dtype)


def _plain_pack(X):
    B, n = X.shape
    nb = -(-n // _BLOCK)
    x = torch.zeros(B, nb * _BLOCK, dtype=torch.float64, device=X.device)
    x[:, :n] = X.to(torch.float64)
    x = x.reshape(B, nb, _BLOCK)
    scales = (x.abs().amax(dim=2) / 127.0).to(torch.float32)
    d = scales.to(torch.float64)[:, :, None]
    q = torch.where(d > 0, torch.round(x / torch.where(d > 0, d, torch.ones_like(d))), torch.zeros_like(x))
    return q.clamp(-127, 127).to(torch.int8).reshape(B, nb * _BLOCK)[:, :n].contiguous(), scales


def _plain_unpack(q, scales, dtype):
    n = q.shape[1]
    return (q.to(torch.float64) * scales.to(torch.float64).repeat_interleave(_BLOCK, dim=1)[:, :n]).to(dtype)


def _highpass(a):
    sign = torch.ones(a.shape[1], dtype=a.dtype, device=a.device)
    sign[1::2] = -1.0
    return a.flip(1) * sign


def _columns(N, half, device):
    """Row r of the low-pass operator has tap j at column (N/2 + 2 r - j) mod 2 half."""
    r = torch.arange(half, device=device)[:, None]
    return (N // 2 + 2 * r - torch.arange(N, device=device)[None, :]) % (2 * half)


def _lines_forward(x, a):
    """x: [E, lines, n], a: [E, N] -> coefficients, and the low-pass levels from n samples down to 2."""
    b, N, n = _highpass(a), a.shape[1], x.shape[2]
    out, levels, cur = torch.empty_like(x), [], x
    while cur.shape[2] > 1:
        half = cur.shape[2] // 2
        at = _columns(N, half, x.device)
        lo = torch.zeros_like(cur[:, :, :half])
        hi = torch.zeros_like(lo)
        for j in range(N):
            v = cur[:, :, at[:, j]]
            lo += a[:, j, None, None] * v
            hi += b[:, j, None, None] * v
        levels.append(cur)
        out[:, :, half:2 * half] = hi
        cur = lo
    out[:, :, :1] = cur[:, :, :1]
    return out, levels


def _lines_backward(d, levels, a):
    """Errors on the coefficients -> errors on the lines, and the gradient [E, N] of the taps."""
    b, N = _highpass(a), a.shape[1]
    grad = torch.zeros_like(a)
    cur = d[:, :, :1]
    for level in reversed(levels):
        half = cur.shape[2]
        dh = d[:, :, half:2 * half]
        at = _columns(N, half, d.device)
        new = torch.zeros_like(level)
        for j in range(N):
            v = level[:, :, at[:, j]]
            grad[:, j] += (cur * v).sum(dim=(1, 2))
            grad[:, N - 1 - j] += (-1.0 if j % 2 else 1.0) * (dh * v).sum(dim=(1, 2))
            new[:, :, at[:, j]] += a[:, j, None, None] * cur + b[:, j, None, None] * dh
        cur = new
    return cur, grad


def _plain_transform(X, a, R, C):
    """Rows, then columns.  X: [E, n] column-major examples."""
    rows, lr = _lines_forward(X.reshape(-1, C, R).transpose(1, 2).contiguous(), a)
    Y, lc = _lines_forward(rows.transpose(1, 2).contiguous(), a)
    return Y.reshape(X.shape), lr, lc


def _plain_forward(X, filters, idx, w, R, C):
    Y = torch.zeros_like(X)
    for j in range(idx.shape[1]):
        Y += w[:, j, None] * _plain_transform(X, filters[idx[:, j].to(torch.int64)], R, C)[0]
    return Y


def _plain_backward(D, X, filters, idx, w, R, C):
    B, k, N = idx.shape[0], idx.shape[1], filters.shape[1]
    dX, dw = torch.zeros_like(D), torch.zeros_like(w)
    grad = torch.zeros(B, k, N, dtype=torch.float64, device=D.device)
    for j in range(k):
        a = filters[idx[:, j].to(torch.int64)]
        Y, lr, lc = _plain_transform(X, a, R, C)
        dw[:, j] = (D * Y).sum(dim=1)
        d, gc = _lines_backward(D.reshape(B, C, R), lc, a)
        d, gr = _lines_backward(d.transpose(1, 2).contiguous(), lr, a)
        dX += w[:, j, None] * d.transpose(1, 2).reshape(B, R * C)
        grad[:, j] = w[:, j, None] * (gc + gr)
    dfilters = torch.zeros_like(filters).index_add_(0, idx.reshape(-1).to(torch.int64), grad.reshape(-1, N))
    return dX, dw, grad, dfilters


# ---- one pass -------------------------------------------------------------------------------------------------

def _routing(case):
    return dict(k=case["k"], score=case["score"], groups=case["groups"], groups_kept=case["kept"],
                renormalise=case["renorm"], scale=case["scale"], score_scale=case["score_scale"])


def _run_own(s, case):
    ctx, kind = s["ctx"], case["kind"]
    if kind == "route":
        v = s["scores"]
        ctx.route(v, case["T"], case["F"], s["idx"], s["w"], bias=s["bias"], counts=s["counts"],
                  row_stride=v.stride(0), col_stride=v.stride(1), **_routing(case))
        return s["idx"], s["w"], s["counts"]
    if kind == "route_grad":
        v = s["scores"]
        ctx.route_backward(v, case["T"], case["F"], s["idx"], s["dw"], s["dscores"], row_stride=v.stride(0),
                           col_stride=v.stride(1), **_routing(case))
        return s["dscores"]
    if kind == "checkpoint":
        ctx.checkpoint_pack(s["X"], case["B"], case["n"], s["q"], s["scales"])
        ctx.checkpoint_unpack(s["q"], s["scales"], case["B"], case["n"], s["out"])
        return s["out"]
    B, R, C, bank = case["B"], case["R"], case["C"], (s["filters"], s["idx"], s["w"])
    if kind == "forward":
        ctx.forward_routed(s["X"], B, R, C, *bank, s["Y"])
        return s["Y"]
    out = []
    if kind == "train":
        ctx.forward_routed(s["X"], B, R, C, *bank, s["Y"], q=s["q"], scales=s["scales"])
        out.append(s["Y"])
    ctx.backprop_routed(s["D"], B, R, C, *bank, s["grad"], q=s["q"], scales=s["scales"], dfilters=s["dfilters"], dw=s["dw"],
                        dX=s["dX"])
    return tuple(out + [s["dX"], s["dw"], s["grad"], s["dfilters"]])


def run(state):
    s, case = state, state["case"]
    if own:
        return _run_own(s, case)
    kind = case["kind"]
    if kind == "route":
        return _plain_route(s["scores"], s["bias"], case)
    if kind == "route_grad":
        return _plain_route_grad(s["scores"], s["idx"], s["dw"], case)
    if kind == "checkpoint":
        return _plain_unpack(*_plain_pack(s["X"]), s["X"].dtype)
    R, C, bank = case["R"], case["C"], (s["filters"], s["idx"], s["w"])
    if kind == "forward":
        return _plain_forward(s["X"], *bank, R, C)
    q, scales = _plain_pack(s["X"]) if kind == "train" else (s["q"], s["scales"])
    back = _plain_backward(s["D"], _plain_unpack(q, scales, torch.float64), *bank, R, C)
    return ((_plain_forward(s["X"], *bank, R, C),) + back) if kind == "train" else back


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("route", "route_grad"):
        T, F, k, e = case["T"], case["F"], case["k"], _BYTES[case["dtype"]]
        if kind == "route":
            b = T * F * e + T * k * 12 + F * 4 + (F * 8 if case["bias"] else 0)
        else:
            # a renormalised weight depends on the chosen scores alone; the whole gradient is written all the same
            b = (T * k * e if case["renorm"] or case["score"] == "sigmoid" else T * F * e) + T * F * e + T * k * 12
        return {"bytes": b, "flops": 4 * T * F}
    if kind == "checkpoint":
        n = case["B"] * case["n"]
        return {"bytes": 2 * n * _BYTES[case["dtype"]], "flops": 4 * n}
    B, n, N, k, F = case["B"], case["R"] * case["C"], case["N"], case["k"], case["F"]
    passes = (case["R"] > 1) + (case["C"] > 1)
    bank = F * N * 8 + B * k * 12
    level = 2 * B * n * N * k * passes          # one operation pair per sample and tap, summed over the levels of a pass
    ckpt = B * (n + 4 * -(-n // _BLOCK))
    forward = {"bytes": B * n * 16 + bank, "flops": 2 * level}
    # low-pass levels once more, the two correlations and the two products that carry the errors on
    backward = {"bytes": B * n * 16 + ckpt + bank + B * k * (8 + 8 * N) + F * N * 8, "flops": 5 * level}
    if kind == "forward":
        return forward
    if kind == "backward":
        return backward
    return {"bytes": forward["bytes"] + backward["bytes"] + ckpt, "flops": forward["flops"] + backward["flops"]}


# ---- the definition in 64 bits, by other means --------------------------------------------------------------------

def _dense_line(a, n):
    """The whole transform of a line as one n x n matrix, and its derivative by every tap: [n, n], [N, n, n]."""
    N = len(a)
    M = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    dM = torch.zeros(N, 1, 1, dtype=torch.float64, device="cuda")
    half = 1
    while 2 * half <= n:
        one = torch.zeros(N, half, 2 * half, dtype=torch.float64, device="cuda")   # tap j of the low-pass operator
        r = torch.arange(half, device="cuda")
        for j in range(N):
            one[j, r, (N // 2 + 2 * r - j) % (2 * half)] += 1.0
        low = torch.zeros(half, 2 * half, dtype=torch.float64, device="cuda")
        high = torch.zeros_like(low)
        dhigh = torch.zeros_like(one)
        for j in range(N):
            low += a[j] * one[j]
            high += (-1.0) ** j * a[N - 1 - j] * one[j]
            dhigh[N - 1 - j] += (-1.0) ** j * one[j]
        dM = torch.cat([torch.stack([dM[j] @ low + M @ one[j] for j in range(N)]), dhigh], dim=1)
        M = torch.cat([M @ low, high], dim=0)
        half *= 2
    return M, dM


def _exact_bank(case, s, X, D, want_y, want_back):
    """Filter by filter: the examples that name it, through dense matrices."""
    B, R, C, N, F, k = (case[x] for x in ("B", "R", "C", "N", "F", "k"))
    f64 = dict(dtype=torch.float64, device="cuda")
    Y, dX = torch.zeros(B, C, R, **f64), torch.zeros(B, C, R, **f64)
    dw, grad, dfilters = torch.zeros(B, k, **f64), torch.zeros(B, k, N, **f64), torch.zeros(F, N, **f64)
    for f in range(F):
        for j in range(k):
            at = torch.nonzero(s["idx"][:, j] == f).reshape(-1)
            if not len(at):
                continue
            MR, dMR = _dense_line([float(v) for v in s["filters"][f]], R)
            MC, dMC = (MR, dMR) if C == R else _dense_line([float(v) for v in s["filters"][f]], C)
            w = s["w"][at, j]
            if want_y:    # an example is held as [C, R]: rows run along C, columns along R
                Y[at] += w[:, None, None] * (MC @ (s["X"].reshape(B, C, R)[at] @ MR.t()))
            if want_back:
                x, d = X.reshape(B, C, R)[at], D.reshape(B, C, R)[at]
                xr, dr = x @ MR.t(), d @ MR
                dw[at, j] = (d * (MC @ xr)).sum(dim=(1, 2))
                dX[at] += w[:, None, None] * (MC.t() @ dr)
                for t in range(N):
                    v = (d * (MC @ (x @ dMR[t].t()))).sum(dim=(1, 2)) + (d * (dMC[t] @ xr)).sum(dim=(1, 2))
                    grad[at, j, t] = w * v
                dfilters[f] += grad[at, j].sum(dim=0)
    n = R * C
    return Y.reshape(B, n), (dX.reshape(B, n), dw, grad, dfilters)


def _exact_rounded(X):
    """Every value replaced by the multiple of its block's scale that is nearest to it."""
    B, n = X.shape
    out = torch.empty(B, n, dtype=torch.float64, device=X.device)
    for at in range(0, n, _BLOCK):
        x = X[:, at:at + _BLOCK].to(torch.float64)
        d = (x.abs().max(dim=1, keepdim=True).values / 127.0).float().double()
        out[:, at:at + _BLOCK] = torch.where(d > 0, torch.clamp(torch.round(x / d), -127.0, 127.0) * d, 0.0 * x)
    return out


def _exact_route(s, case):
    """Row by row choices through one sort of (value, index); weights from logarithms."""
    T, F, k, G = case["T"], case["F"], case["k"], case["groups"]
    v = case["score_scale"] * s["scores"].double()
    logp = v - torch.logsumexp(v, 1, keepdim=True) if case["score"] == "softmax" else -torch.log1p(torch.exp(-v))
    c = v if s["bias"] is None else torch.exp(logp) + s["bias"]
    if case["kept"] < G:
        per = (torch.exp(logp) if s["bias"] is None else c).reshape(T * G, F // G)
        first = per.max(dim=1).values
        rest = per.clone()
        rest[torch.arange(T * G, device=v.device), per.max(dim=1).indices] = -math.inf
        second = rest.max(dim=1).values
        score = (first + torch.where(second > -math.inf, second, torch.zeros_like(second))).reshape(T, G)
        beats = (score[:, None, :] > score[:, :, None]).sum(dim=2)
        i = torch.arange(G, device=v.device)
        beats += ((score[:, None, :] == score[:, :, None]) & (i[None, None, :] < i[None, :, None])).sum(dim=2)
        c = c.masked_fill((beats >= case["kept"]).repeat_interleave(F // G, dim=1), -math.inf)
    idx = torch.full((T, k), -1, dtype=torch.int64, device=v.device)
    for j in range(k):
        m = c.max(dim=1, keepdim=True).values
        at = (c == m).to(torch.int8).argmax(dim=1)
        hit = m[:, 0] > -math.inf
        idx[:, j] = torch.where(hit, at, idx[:, j])
        c = c.scatter(1, at[:, None], -math.inf)
    lw = logp.gather(1, idx.clamp(min=0)).masked_fill(idx < 0, -math.inf)
    if case["renorm"]:
        lw = lw - torch.logsumexp(lw, 1, keepdim=True)
    counts = torch.bincount(idx[idx >= 0], minlength=F).to(torch.int32)
    return idx.to(torch.int32), case["scale"] * torch.exp(lw), counts


def _exact_route_grad(s, case):
    """Through the Jacobian of the weights, one chosen filter at a time."""
    v = case["score_scale"] * s["scores"].double()
    idx = s["idx"].long()
    hot = torch.zeros_like(v)
    out = torch.zeros_like(v)
    if case["score"] == "softmax":
        logp = v - torch.logsumexp(v, 1, keepdim=True)
    else:
        logp = -torch.log1p(torch.exp(-v))
    q = torch.exp(-torch.log1p(torch.exp(v)))                         # 1 - sigmoid
    lw = logp.gather(1, idx.clamp(min=0)).masked_fill(idx < 0, -math.inf)
    if case["renorm"]:
        lw = lw - torch.logsumexp(lw, 1, keepdim=True)
    w = torch.exp(lw)
    mean = (w * s["dw"]).sum(dim=1)                                    # d/d log p of a renormalised weight subtracts this
    for j in range(idx.shape[1]):
        live = idx[:, j] >= 0
        at = idx[:, j].clamp(min=0)[:, None]
        dlog = (w[:, j] * (s["dw"][:, j] - (mean if case["renorm"] else 0.0))).masked_fill(~live, 0.0)[:, None]
        if case["score"] == "softmax":
            hot = hot.scatter_add(1, at, dlog)
        else:
            hot = hot.scatter_add(1, at, dlog * q.gather(1, at))
    out = hot
    if case["score"] == "softmax" and not case["renorm"]:
        out = hot - torch.exp(logp) * hot.sum(dim=1, keepdim=True)
    return out * (case["scale"] * case["score_scale"])


def exact(case, seed):
    kind = case["kind"]
    if kind not in ("route", "route_grad", "checkpoint"):
        n = max(case["R"], case["C"])
        # multiplications of building the matrices and of the products with them
        if case["F"] * case["N"] * n ** 3 + case["B"] * case["k"] * case["N"] * case["R"] * case["C"] * n > 4e13:
            return None
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if kind == "route":
        return _exact_route(s, case)
    if kind == "route_grad":
        return _exact_route_grad(s, case)
    if kind == "checkpoint":
        return _exact_rounded(s["X"])
    if kind == "forward":
        return _exact_bank(case, s, None, None, True, False)[0]
    if kind == "backward":
        scales = s["scales"].double()
        X = torch.stack([s["q"][:, i].double() * scales[:, i // _BLOCK] for i in range(s["q"].shape[1])], dim=1)
        return _exact_bank(case, s, X, s["D"], False, True)[1]
    Y, back = _exact_bank(case, s, _exact_rounded(s["X"]), s["D"], True, True)
    return (Y,) + back
