"""Plain 64-bit implementations of the order by expert, of the sums of sorted rows
and of products with 4-bit matrices, from their definitions (numpy, on the CPU)."""
import numpy as np

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative to the value
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}  # the least step


def order(ids, E):
    """(rows, positions, experts, offsets) by (expert, entry)."""
    n, k = ids.shape
    flat = ids.reshape(-1)
    held = [(int(e), i) for i, e in enumerate(flat) if 0 <= e < E]
    held.sort()
    rows, experts = np.full(n * k, -1, np.int32), np.full(n * k, -1, np.int32)
    pos = np.full(n * k, -1, np.int32)
    for p, (e, i) in enumerate(held):
        rows[p], experts[p], pos[i] = i, e, p
    offsets = np.array([sum(1 for e, _ in held if e < x) for x in range(E + 1)], np.int32) if len(held) * E < 4e6 else \
        np.concatenate([[0], np.cumsum(np.bincount([e for e, _ in held], minlength=E)[:E])]).astype(np.int32)
    return rows, pos.reshape(n, k), experts, offsets


def gather(x, rows, k):
    out = np.zeros((rows.size, x.shape[1]), x.dtype)
    live = rows >= 0
    out[live] = x[rows[live] // k]
    return out


def picks(y, pos):
    """y's rows by (token, pick), 0 without one."""
    return np.where((pos >= 0)[..., None], y[np.maximum(pos, 0)], 0.0)


def combine(y, pos, w, shared=None):
    """(sums, sums of magnitudes)"""
    w = np.where(pos >= 0, np.ones_like(pos, np.float64) if w is None else w, 0.0)
    v = picks(y, pos) * w[..., None]
    s, mag = v.sum(1), np.abs(v).sum(1)
    return (s, mag) if shared is None else (s + shared, mag + np.abs(shared))


def combine_tol(s, mag, k, t):
    """A product or sum of 32 bits rounds by 2^-24 of at most the magnitudes' sum: k products (fused or not) and k
    sums with the shared row's; 2^-149 each where they underflow; then one rounding to t."""
    return 1.01 * ((2 * k + 1) * 2.0 ** -24 * mag + (2 * k + 1) * 2.0 ** -149 + HALF[t] * np.abs(s) + TINY[t])


def w4_values(codes, scales, zeros, K, group):
    """uint8 [..., rows, ceil(K / 2)], f64 [..., rows, n], zeros or None -> f64 [..., rows, K]: scale (code - zero), and
    |scale| (code + zero)"""
    q = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)[..., :K].astype(np.float64)
    at = np.arange(K) // group
    z = 8.0 if zeros is None else zeros[..., at].astype(np.float64)
    return (q - z) * scales[..., at], (q + z) * np.abs(scales[..., at])


def w4_tol(mag, K):
    """Of sum s (q - z) x, computed as the sum over groups of s (sum q x) - s z (sum x); mag = the sum of |s| (q + z) |x|,
    which bounds every partial sum. Each of the up to 128 additions of two tiles, on the tensor cores, may cut off 2^-23 of at
    most mag. Every tile's scale and every group's s z (two roundings) are applied with a rounding each, 2^-24; so are the
    sums of a stage, of up to 8 warps and 8 CTAs, of 2 planes and the bias (20), and the sums of x over a group
    (8 levels). A 32-bit x is held to 2^-22 of its value. What lies more than 2^24 below the largest x of its 256 values is
    cut off at 2^-39 of that: the largest is one of mag's, times at most 30 / 1 between (q + z) of two places,
    hence 256 * 30 * 2^-39 < 2^-26 of mag."""
    return 1.01 * mag * (128 * 2.0 ** -23 + (K / 64 + 3 * (K / 32 + 1) + K / 256 + 20 + 8 + 2) * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -26) + 1e-36


def glu(op, g, u, limit=0.0):
    with np.errstate(over="ignore"):
        sig = lambda v: 1.0 / (1.0 + np.exp(-v))   # noqa: E731
        if op == 0:
            return u * g * sig(g)
        if op == 1:
            return u * 0.5 * g * (1.0 + np.tanh(np.sqrt(2 / np.pi) * g * (1.0 + 0.044715 * g * g)))
        if op == 2:
            x = np.minimum(g, 7.0)
            return x * sig(1.702 * x) * (np.clip(u, -7.0, 7.0) + 1.0)
        if op == 3:
            x = np.minimum(g, limit)
            return x * sig(x) * np.clip(u, -limit, limit)
        return u * g


def glu_tol(op, g, u, eg, eu, limit=0.0):
    """What errors eg and eu of the arguments do (the slopes of the gates' curves are below 1.2, of geglu's below
    1.2 as well, and 1.702 x sigma' + sigma below 1.2; that of the product is the other factor), then the GLU's own
    roundings: exp, the quotient, the sums and products are within 16 units of 2^-24, exp's argument of op 2 within
    2 |1.702 g| more; geglu's tanh near -1 leaves an absolute error of 2^-22 |g u|."""
    v = np.abs(glu(op, g, u, limit))
    cap = {2: 7.0, 3: limit}.get(op)
    gm, um = np.abs(g) + eg, np.abs(u) + eu
    if cap is not None:
        um = np.minimum(um, cap)
    uf = um + 1.0 if op == 2 else um
    slope = 1.2 * eg * uf + 1.2 * eu * gm
    return slope + v * (16 + 4 * gm) * 2.0 ** -24 + gm * uf * 2.0 ** -22 * (op == 1) + 2.0 ** -100


# Of products with codes and zeros even over 0..15 (or no zeros) and x N(0, 1), relative, in the 2-norm over many outputs. A
# chain of up to 8 tensor-core sums cuts off up to 2^-23 of each partial sum, half of it in the mean; the i-th has
# sqrt(i / 8) of the last one's rms, so all in the same direction 6.1 * 2^-24 = 3.7e-7 of sums of q x, whose rms is 8.8 for the
# 4.6 or more of (q - z) x: 6.9e-7. A 32-bit x is held to 2^-22, 1.4e-7 rms. The 32-bit roundings behind the tensor cores (a
# scale, a zero, stages, warps, CTAs, passes, sums of x: 40 in a chain at most) are off by 2^-24 / sqrt(3) rms each, at
# random: sqrt(40) * 3.4e-8 * 1.9 = 4.2e-7. Together 1.1e-6.
W4_NORM = 1.5e-6
