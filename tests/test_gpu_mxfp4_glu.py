"""The GLU of the MXFP4 product, apart from its sums: blocks whose products and
sums are exact in 32 bits in any order, so that what differs is the GLU."""
import numpy as np
import pytest
import torch

import mx_ref as R

pytestmark = pytest.mark.gpu

LIMIT = 1.25


def _exact_case(rng, n, k, E, K, rows, shift):
    """Codes of one scale: x (one plane holds it) in multiples of 0.5 up to 6, matrices the same times 2^-shift:
    sums of multiples of 2^-(2 + shift) that stay below 36 K x 4 <= 2^19 of these steps for K <= 2048, so every
    order of additions is exact."""
    def codes(*shape):
        c = rng.integers(0, 16, size=shape, dtype=np.uint8)
        c[..., ::32] |= 7                                  # every block has a 6: its scale is 2^0
        return c.reshape(*shape[:-1], -1, 32)
    c = codes(n, K)
    x = (R.E2M1[c & 7] * np.where(c & 8, -1, 1)).reshape(n, K)
    W = [R.to_blocks(np.full((E, rows, K // 32), 127 - shift, np.uint8), codes(E, rows, K)) for _ in range(2)]
    ids = np.argsort(rng.normal(size=(n, E)), axis=1)[:, :k].astype(np.int32)
    return x.astype(np.float32), W, ids


def _call(pkg, cuda, x, W, ids, op, bias=(None, None)):
    t = lambda a: None if a is None else torch.from_numpy(a).to(cuda)   # noqa: E731
    up, gate = (pkg.MXFP4Weights(t(b), x.shape[1], b.shape[1]) for b in W)
    y = pkg.mxfp4_mul_mat_id(up, t(x), t(ids), gate=gate, bias=t(bias[0]), gate_bias=t(bias[1]), glu_op=op, glu_limit=LIMIT,
                             planes=1)
    assert pkg.moe_cache.device_error() == 0
    return y.cpu().numpy()


@pytest.mark.parametrize("op", [0, 1, 2, 3, 4])
def test_a_token_alone_and_in_a_batch(pkg, cuda, op):
    """One token's outputs are the same bits however many tokens share the call: the sums are exact here, and one
    GLU serves the forms that share K over a cluster and those that do not."""
    rng = np.random.default_rng(op)
    x, W, ids = _exact_case(rng, 1, 4, 8, 2048, 256, 6)
    bias = tuple(rng.normal(size=(8, 256)).astype(np.float32) for _ in range(2))
    one = _call(pkg, cuda, x, W, ids, op, bias)
    for n in (2, 16, 30, 100, 700):
        many = _call(pkg, cuda, np.repeat(x, n, 0), W, np.repeat(ids, n, 0), op, bias)
        for t in (0, n // 2, n - 1):
            np.testing.assert_array_equal(many[t], one[0])


@pytest.mark.parametrize("op", [0, 2, 3])
@pytest.mark.parametrize("n", [1, 9, 40, 260])
def test_rounding_of_the_glu(pkg, cuda, op, n):
    """With exact sums the error is the GLU's, in units of 2^-24 of the value: exp is off by one unit of its last
    place (2 of them), the quotient by two (4), 1 + e and the product by a rounding each -- 8, 9 allowed for their
    products -- and in the clamped form of op 2 also u + 1 by a rounding and the argument t = 1.702 g, whose constant
    and product are off by 2^-24 each: 2 |t| more. Below that, the approximate quotient x / d is defined to be 0
    for d above 2^126, where it is less than |x| 2^-126; its factor is u, or u clamped to [-7, 7] plus 1: at most
    |x| (|u| + 1) 2^-126, and |x| <= |g| + 7."""
    rng = np.random.default_rng(n)
    x, W, ids = _exact_case(rng, n, 4, 8, 512, 130, 4)
    y = _call(pkg, cuda, x, W, ids, op)
    u, _ = R.product(W[0], x, ids, 1)
    g, _ = R.product(W[1], x, ids, 1)
    assert np.abs(g).max() > 15
    ref = R.glu(op, g, u, LIMIT)
    units = 9 + (1 + 2 * 1.702 * np.abs(g) if op == 2 else 0)
    assert (np.abs(y - ref) <= units * 2.0 ** -24 * np.abs(ref) + (np.abs(g) + 7) * (np.abs(u) + 1) * 2.0 ** -126).all()


@pytest.mark.parametrize("op", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("n", [1, 9, 40, 260])
def test_nan_passes_the_clamps(pkg, cuda, op, n):
    """A NaN of x, of a gate row or of an up row is a NaN of the outputs it enters, and of no other."""
    rng = np.random.default_rng(n)
    E, k, K, rows = 8, 4, 512, 130
    x, W, ids = _exact_case(rng, n, k, E, K, rows, 4)
    clean = _call(pkg, cuda, x, W, ids, op)
    x[n // 2, 77] = np.nan
    W[0][ids[0, 0], 3, 17] = 255          # a NaN scale in an up row,
    W[1][ids[0, 0], 5, 34] = 255          # and in a gate row, of one expert
    want = np.zeros((n, k, rows), bool)
    want[n // 2] = True
    hit = ids == ids[0, 0]
    want[..., 3] |= hit
    want[..., 5] |= hit
    y = _call(pkg, cuda, x, W, ids, op)
    assert np.isnan(y[want]).all()
    np.testing.assert_array_equal(y[~want], clean[~want])
