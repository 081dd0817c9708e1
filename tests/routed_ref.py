"""Plain 64-bit forms of the routed filter bank's operators, from their definitions in include/wavenet_hip.h."""
import numpy as np

BLOCK = 64


def shares(s, score):
    """p of every filter; closed filters (s = -inf) have none."""
    with np.errstate(over="ignore", invalid="ignore"):
        if score == "softmax":
            top = s.max(axis=1, keepdims=True)
            e = np.where(s > -np.inf, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
            z = e.sum(axis=1, keepdims=True)
            return np.where(z > 0, e / np.where(z > 0, z, 1.0), 0.0)
        return 1.0 / (1.0 + np.exp(-s))


def route(scores, k, score="softmax", bias=None, groups=1, groups_kept=None, renormalise=True, scale=1.0, score_scale=1.0):
    s = np.asarray(scores, dtype=np.float64) * score_scale
    T, F = s.shape
    kept = groups if groups_kept is None else groups_kept
    void = ~(s < np.inf).all(axis=1)
    s = np.where(void[:, None], -np.inf, s)
    p = shares(s, score)
    c = s.copy() if bias is None else p + bias
    c[~(c > -np.inf) | (s == -np.inf)] = -np.inf
    idx = np.full((T, k), -1, dtype=np.int32)
    w = np.zeros((T, k))
    per = F // groups
    for t in range(T):
        row = c[t].copy()
        if kept < groups:
            of = np.where(row > -np.inf, p[t] if bias is None else row, -np.inf).reshape(groups, per)
            best = np.sort(of, axis=1)[:, ::-1][:, :2]
            gs = [b[b > -np.inf].sum() if (b > -np.inf).any() else -np.inf for b in best]
            order = sorted(range(groups), key=lambda g: (-gs[g], g))[:kept]
            for g in range(groups):
                if g not in order:
                    row[g * per:(g + 1) * per] = -np.inf
        order = sorted(range(F), key=lambda f: (-row[f], f))[:k]
        chosen = [f for f in order if row[f] > -np.inf]
        idx[t, :len(chosen)] = chosen
        q = p[t, chosen]
        if renormalise and len(chosen):
            if q.sum() > 1e-280:
                q = q / q.sum()
            else:                        # shares too small for a double: from their logarithms
                lp = s[t, chosen] if score == "softmax" else np.minimum(s[t, chosen], 0) - np.log1p(np.exp(-np.abs(s[t, chosen])))
                q = np.exp(lp - lp.max())
                q = q / q.sum()
        w[t, :len(chosen)] = scale * q
        if void[t]:
            w[t] = np.nan
    counts = np.bincount(idx[idx >= 0], minlength=F).astype(np.int32)
    return idx, w, counts


def route_backward(scores, idx, dw, score="softmax", renormalise=True, scale=1.0, score_scale=1.0):
    """Through the Jacobian of the weights, row by row."""
    s = np.asarray(scores, dtype=np.float64) * score_scale
    T, F = s.shape
    p = shares(s, score)
    out = np.zeros((T, F))
    for t in range(T):
        at = [j for j in range(idx.shape[1]) if 0 <= idx[t, j] < F]
        if not at:
            continue
        f = idx[t, at]
        g = scale * dw[t, at]
        q = p[t, f]
        if score == "softmax":
            J = -np.outer(q, p[t])
            J[np.arange(len(f)), f] += q
        else:
            J = np.zeros((len(f), F))
            J[np.arange(len(f)), f] = q / (1.0 + np.exp(s[t, f]))
        if renormalise:
            z = q.sum()
            J = J / z - np.outer(q, J.sum(axis=0)) / z ** 2
        out[t] = score_scale * (g @ J)
    return out


def pack(X):
    X = np.asarray(X, dtype=np.float64)
    B, n = X.shape
    nb = -(-n // BLOCK)
    q = np.zeros((B, n), dtype=np.int8)
    scales = np.zeros((B, nb), dtype=np.float32)
    with np.errstate(all="ignore"):
        for i in range(nb):
            x = X[:, i * BLOCK:(i + 1) * BLOCK]
            m = np.where(np.isfinite(x), np.abs(x), np.nan).max(axis=1)
            scales[:, i] = (m / 127.0).astype(np.float32)
            d = scales[:, i].astype(np.float64)[:, None]
            v = np.clip(np.rint(x / d), -127, 127)
            q[:, i * BLOCK:(i + 1) * BLOCK] = np.where(np.isfinite(d) & (d > 0), v, 0).astype(np.int8)
    return q, scales


def unpack(q, scales):
    with np.errstate(invalid="ignore"):
        return q.astype(np.float64) * np.repeat(scales.astype(np.float64), BLOCK, axis=1)[:, :q.shape[1]]


def forward(oracle, X, filters, idx, w):
    """X: [B, R, C]; entries that name no filter add 0 * w."""
    Y = np.zeros(X.shape)
    for e in range(len(X)):
        for j in range(idx.shape[1]):
            if 0 <= idx[e, j] < len(filters):
                Y[e] += w[e, j] * oracle.band_forward_2d(filters[idx[e, j]], X[e])[3]
            else:
                Y[e] += 0.0 * w[e, j]
    return Y


def backward(oracle, D, X, filters, idx, w):
    B, k, N = idx.shape[0], idx.shape[1], filters.shape[1]
    grad, dw, dX = np.zeros((B, k, N)), np.zeros((B, k)), np.zeros(X.shape)
    dfilters = np.zeros(filters.shape)
    for e in range(B):
        for j in range(k):
            f = idx[e, j]
            if not 0 <= f < len(filters):
                dX[e] += 0.0 * w[e, j]
                continue
            a = filters[f]
            Pr, Y1, Pc, Y = oracle.band_forward_2d(a, X[e])
            grad[e, j] = w[e, j] * oracle.band_backprop_2d(a, D[e], X[e], Pr, Y1, Pc)
            dw[e, j] = (D[e] * Y).sum()
            dX[e] += w[e, j] * oracle.band_inverse_2d(a, D[e])      # the inverse is the transpose of the cascade
            dfilters[f] += grad[e, j]
    return grad, dfilters, dw, dX
