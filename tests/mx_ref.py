"""Plain 64-bit implementations of the MXFP4 path and the router, from their
definitions (numpy, on the CPU)."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
MIN_SUM = 2.0 ** -14


def quantize_plane(x):
    """x f64 [..., K] -> (scale bytes uint8 [..., K/32], codes uint8 [..., K/32, 32]): nearest, ties to the even code."""
    x = np.asarray(x, dtype=np.float64)
    v = x.reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    amax = np.abs(v).max(-1)
    _, e = np.frexp(amax)
    e = np.where(amax == 0, -127, np.maximum(e - 3, -127))
    mag = np.abs(v) / np.exp2(e.astype(np.float64))[..., None]
    dist = np.abs(mag[..., None] - E2M1)
    best = dist.min(-1, keepdims=True)
    near = dist == best
    code = np.where(near, np.arange(8) + 10 * (np.arange(8) % 2), 99).argmin(-1)   # an even code before an odd one
    code = np.where(mag > 6, 7, code).astype(np.uint8)
    code |= (np.signbit(v).astype(np.uint8) << 3)
    code[bad] = 0
    return np.where(bad, 255, e + 127).astype(np.uint8), code


def to_blocks(scale, code):
    b = np.empty(scale.shape + (17,), dtype=np.uint8)
    b[..., 0] = scale
    b[..., 1:] = code[..., :16] | (code[..., 16:] << 4)
    return b.reshape(*scale.shape[:-1], -1)


def from_blocks(blocks, K):
    """uint8 [..., 17 K / 32] -> f64 [..., K]."""
    b = blocks.reshape(*blocks.shape[:-1], K // 32, 17)
    c = np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
    v = np.where(c & 8, -1.0, 1.0) * E2M1[c & 7]
    s = np.where(b[..., :1] == 255, np.nan, np.exp2(b[..., :1].astype(np.float64) - 127))
    return (v * s).reshape(*blocks.shape[:-1], K)


def quantize(x, planes=1):
    """f64 [..., K] -> list of uint8 blocks, one per plane."""
    left, out = np.asarray(x, dtype=np.float64), []
    for _ in range(planes):
        out.append(to_blocks(*quantize_plane(left)))
        left = left - from_blocks(out[-1], left.shape[-1])
    return out


def values(x, planes=1):
    x = np.asarray(x, dtype=np.float64)
    return sum(from_blocks(b, x.shape[-1]) for b in quantize(x, planes))


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-x))


def glu(op, g, u, limit=0.0):
    g, u = np.asarray(g, np.float64), np.asarray(u, np.float64)
    if op == 0:
        return u * g * sigmoid(g)
    if op == 1:
        return u * 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * g * (1 + 0.044715 * g * g)))
    if op == 2:
        x = np.minimum(g, 7.0)
        return x * sigmoid(1.702 * x) * (np.clip(u, -7, 7) + 1)
    if op == 3:
        x = np.minimum(g, limit)
        return x * sigmoid(x) * np.clip(u, -limit, limit)
    return u * g


def product(W, x, ids, planes, bias=None):
    """W blocks uint8 [E, rows, bytes], x [n, K] or [n, k, K], ids [n, k] ->
    (y f64 [n, k, rows], the sums of the terms' magnitudes); picks outside the experts give NaN."""
    n, k = ids.shape
    K = x.shape[-1]
    X = values(x, planes)
    y = np.full((n, k, W.shape[1]), np.nan)
    mag = np.zeros_like(y)
    M = {e: from_blocks(W[e], K) for e in np.unique(ids) if 0 <= e < W.shape[0]}
    for t in range(n):
        for p in range(k):
            e = ids[t, p]
            if e in M:
                row = X[t, p] if x.ndim == 3 else X[t]
                y[t, p] = M[e] @ row
                mag[t, p] = np.abs(M[e]) @ np.abs(row)
                if bias is not None:
                    y[t, p] += bias[e]
                    mag[t, p] += np.abs(bias[e])
    return y, mag


def product_tol(mag, K, planes):
    """Bound on the error of a product: every K = 64 step of a plane (and every cluster rank, at most 8, and the
    bias) is one 32-bit addition that may lose a unit of the last place, 2^-23, of a sum no larger than the
    terms' magnitudes together."""
    return ((-(-K // 64) * planes) + 9) * 2.0 ** -23 * mag


def route(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_score="top2", norm_w=False, scale=1.0):
    """(ids [n, k], weights f64 [n, k])."""
    l = np.asarray(logits, dtype=np.float64)
    l = np.where(np.isnan(l), -np.inf, np.minimum(l, np.finfo(np.float32).max))
    n, E = l.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        if score == "softmax":
            m = l.max(1, keepdims=True)
            s = np.where(np.isfinite(l), np.exp(l - np.where(np.isfinite(m), m, 0)), 0.0)
            s = s / np.where(s.sum(1, keepdims=True) == 0, 1, s.sum(1, keepdims=True))
        elif score == "sigmoid":
            s = sigmoid(l)
        else:
            s = l
        c = s + (0 if bias is None else np.asarray(bias, dtype=np.float64)[None])
        if bias is None and n_group == 1:
            c = l
    c = np.where(np.isneginf(l) | np.isnan(c), -np.inf, c)
    ids = np.zeros((n, k), dtype=np.int32)
    w = np.zeros((n, k))
    size = E // n_group
    for t in range(n):
        r = c[t].copy()
        if n_group > 1:
            worth = []
            for g in range(n_group):
                v = np.sort(r[g * size: (g + 1) * size])[::-1]
                worth.append(v[0] if group_score == "max" or size == 1 or np.isneginf(v[1]) else v[0] + v[1])
            best = sorted(range(n_group), key=lambda g: (-worth[g], g))[:topk_group]
            for g in range(n_group):
                if g not in best:
                    r[g * size: (g + 1) * size] = -np.inf
        ids[t] = sorted(range(E), key=lambda e: (-r[e], e))[:k]
        live = r[ids[t]] > -np.inf
        if score == "softmax_topk":
            if live.any():
                v = l[t, ids[t]]
                x = np.where(live, np.exp(v - v[live].max()), 0.0)
                w[t] = x / x.sum()
        else:
            w[t] = np.where(live, s[t, ids[t]], 0.0)
        if norm_w:
            w[t] = w[t] / max(w[t].sum(), MIN_SUM)
    return ids, w * scale
