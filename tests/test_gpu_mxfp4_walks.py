"""How the MXFP4 product walks its work: every chunk width with and without a
gate, with K shared by a cluster, and with more tiles than CTAs, so that the
ring and both accumulator sets are carried from item to item. Values against the
64-bit reference (mx_ref)."""
import numpy as np
import pytest
import torch

import mx_ref as R

pytestmark = pytest.mark.gpu


def _experts(rng, E, rows, K):
    b = rng.integers(0, 256, size=(E, rows, K // 32, 17), dtype=np.uint8)
    b[..., 0] = rng.integers(116, 122, size=b.shape[:-1])
    return b.reshape(E, rows, -1)


@pytest.mark.parametrize("glu", [None, 0, 2])
@pytest.mark.parametrize("n,k,E,K,rows,per_pick,planes", [
    # up to 64 picks, rows quantised by the product: up to 1024 tiles for 296 CTAs,
    (8, 8, 64, 768, 2048, True, 2),
    (8, 8, 64, 768, 2048, False, 2),
    (16, 4, 16, 1024, 3000, False, 1),     # chunks of several rows,
    (13, 4, 52, 1440, 1000, False, 2),     # and padded tiles
    # 16 columns
    (33, 4, 32, 512, 700, False, 2),
    (40, 2, 64, 1024, 100, True, 2),       # K shared
    (300, 2, 128, 256, 600, False, 1),     # more tiles than CTAs
    # 64 columns
    (100, 4, 16, 384, 250, True, 2),
    (40, 2, 4, 1024, 128, False, 2),       # K shared
    (250, 4, 40, 256, 1024, False, 2),     # more tiles than CTAs
    (250, 4, 24, 416, 1000, False, 1),
    # 96 with a gate, 192 without
    (300, 4, 4, 352, 250, True, 2),
    (512, 8, 16, 256, 1024, False, 2),     # more tiles than CTAs
    (700, 3, 7, 416, 1500, False, 1),
])
def test_walk(pkg, cuda, n, k, E, K, rows, per_pick, planes, glu):
    """Tolerances as in the product's other tests: mx_ref.product_tol for the sums; with a GLU their errors
    times its slopes (1.13 |u| + 8.5 by g, |g| + 1 by u), plus 3e-6 of its factors."""
    rng = np.random.default_rng(n + K)
    U, G = _experts(rng, E, rows, K), _experts(rng, E, rows, K)
    x = rng.normal(size=(n, k, K) if per_pick else (n, K)).astype(np.float32)
    # skewed, as routers pick: some experts fill several chunks, some none
    ids = np.argsort(1.1 * np.log(rng.permutation(E) + 1.0) - rng.normal(size=(n, E)), axis=1)[:, :k].astype(np.int32)
    bu, bg = (rng.normal(size=(E, rows)).astype(np.float32) for _ in range(2))
    t = lambda a: torch.from_numpy(a).to(cuda)   # noqa: E731
    wu, wg = (pkg.MXFP4Weights(t(b), K, rows) for b in (U, G))
    kw = {} if glu is None else dict(gate=wg, gate_bias=t(bg), glu_op=glu)
    y = pkg.mxfp4_mul_mat_id(wu, t(x), t(ids), bias=t(bu), planes=planes, **kw)
    again = pkg.mxfp4_mul_mat_id(wu, t(x), t(ids), bias=t(bu), planes=planes, **kw)
    assert pkg.moe_cache.device_error() == 0 and torch.equal(y, again)
    y = y.cpu().numpy()
    u, mu = R.product(U, x, ids, planes, bu)
    du = R.product_tol(mu, K, planes)
    if glu is None:
        assert (np.abs(y - u) <= du).all()
        return
    g, mg = R.product(G, x, ids, planes, bg)
    dg = R.product_tol(mg, K, planes)
    tol = (1.13 * np.abs(u) + 8.5) * dg + (np.abs(g) + 1) * du + 3e-6 * (np.abs(g) + 1) * (np.abs(u) + 1)
    assert (np.abs(y - R.glu(glu, g, u)) <= tol).all()
