"""Routing (moe_b200_route_experts) against the 64-bit reference: ids exactly,
weights to the error of their 32-bit steps.

Weights: exp to 2 ulp (2^-22), one rounding each of 1 + e and the quotient
(sigmoid), for softmax the rounding of l - max (at most |l - max| 2^-24, below
2^-19 for the logits here) and up to 37 + 5 additions; a sum over the picks, a
quotient and a product more with norm_w and scale: below 5e-6 of the weight."""
import numpy as np
import pytest
import torch

import mx_ref as R
from moe_data import zipf_logits

pytestmark = pytest.mark.gpu

RTOL = 5e-6
SCORES = ("softmax", "sigmoid", "softmax_topk")


def _check(pkg, cuda, logits, k, dtype=torch.float32, bias=None, **kw):
    lg = torch.from_numpy(np.asarray(logits, dtype=np.float32)).to(cuda).to(dtype)
    bt = None if bias is None else torch.from_numpy(np.asarray(bias, dtype=np.float32)).to(cuda)
    ids, w = pkg.route_experts(lg, k, bias=bt, **kw)
    rid, rw = R.route(lg.float().cpu().numpy(), k, bias=None if bias is None else np.asarray(bias, np.float32), **kw)
    np.testing.assert_array_equal(ids.cpu().numpy(), rid)
    np.testing.assert_allclose(w.cpu().numpy(), rw, rtol=RTOL, atol=1e-37)
    return ids, w


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("n_tok,E,k,bias,n_group,topk_group,group_score,norm_w,scale", [
    (1, 1, 1, False, 1, 1, "max", False, 1.0),
    (1, 256, 8, True, 8, 4, "top2", True, 2.5),
    (5, 40, 32, True, 1, 1, "max", True, 1.0),
    (33, 160, 6, False, 8, 3, "max", False, 1.0),
    (64, 256, 8, True, 8, 4, "top2", True, 2.5),
    (130, 96, 5, True, 3, 2, "top2", False, 1.5),       # groups whose number is not a power of two
    (17, 320, 16, False, 32, 4, "top2", True, 1.0),     # 32 groups of 10
    (9, 512, 8, True, 1, 1, "max", False, 1.0),
    (7, 1000, 31, True, 4, 4, "top2", True, 1.0),       # every group stays
    (3, 1024, 32, False, 1, 1, "max", False, 1.0),
    (11, 24, 4, True, 24, 6, "top2", False, 1.0),       # groups of one expert
])
def test_route(pkg, cuda, score, n_tok, E, k, bias, n_group, topk_group, group_score, norm_w, scale):
    rng = np.random.default_rng(E + k)
    b = 0.1 * rng.normal(size=E) if bias else None
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _check(pkg, cuda, zipf_logits(n_tok, E, seed=E + n_tok), k, dtype, b, score=score, n_group=n_group, topk_group=topk_group,
               group_score=group_score, norm_w=norm_w, scale=scale)


def test_route_long_batch(pkg, cuda):
    E = 256
    b = 0.1 * np.random.default_rng(3).normal(size=E)
    _check(pkg, cuda, zipf_logits(4099, E, seed=3), 8, bias=b, score="sigmoid", n_group=8, topk_group=4, norm_w=True, scale=2.5)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("n_group,topk_group", [(1, 1), (4, 2)])
def test_ties_and_close_pairs(pkg, cuda, score, n_group, topk_group):
    """Equal scores go to the lower id (groups too); scores that 32 bits cannot tell apart go by 64 bits."""
    rng = np.random.default_rng(7)
    E, n, k = 64, 96, 9
    kw = dict(score=score, n_group=n_group, topk_group=topk_group, group_score="top2")
    flat = np.zeros((n, E), np.float32)
    _check(pkg, cuda, flat, k, **kw)
    _check(pkg, cuda, flat, k, bias=np.zeros(E), **kw)
    steps = np.round(rng.normal(size=(n, E)) * 4) / 4
    _check(pkg, cuda, steps, k, **kw)
    _check(pkg, cuda, steps, k, bias=np.round(rng.normal(size=E)) / 8, **kw)
    near = (0.5 + 2e-7 * rng.integers(-4, 5, size=(n, E))).astype(np.float32)
    _check(pkg, cuda, near, k, bias=1e-8 * rng.integers(-9, 10, size=E), **kw)
    cancel = rng.normal(size=E).astype(np.float32)                   # logits whose scores the bias levels
    lv = R.route(cancel[None], E, score=score)[1] if score != "softmax_topk" else None
    if lv is not None:
        s = np.empty(E)
        s[R.route(cancel[None], E, score=score)[0][0]] = lv[0]
        _check(pkg, cuda, np.tile(cancel, (n, 1)), k, bias=-s, **kw)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n_group,topk_group", [(1, 1), (4, 2)])
def test_masked_logits(pkg, cuda, score, bias, n_group, topk_group):
    E, k = 32, 6
    rng = np.random.default_rng(11)
    l = rng.normal(size=(12, E)).astype(np.float32)
    l[0] = -np.inf                            # nothing left
    l[1] = np.nan
    l[2, :] = -np.inf
    l[2, 17] = 0.5                            # one expert
    l[3, ::2] = -np.inf
    l[4, 5] = np.nan                          # a NaN in a masked place
    l[5, 9] = np.inf
    l[6, [3, 30]] = np.inf
    l[7] = np.finfo(np.float32).min           # a mask of the type's lowest value everywhere
    l[8, :20] = np.finfo(np.float32).min
    l[9] = 88.0
    l[10] = -104.0                            # exp overflows / underflows
    b = (0.1 * rng.normal(size=E)) if bias else None
    if bias:
        b[7], b[8] = -np.inf, np.nan
    ids, w = _check(pkg, cuda, l, k, bias=b, score=score, n_group=n_group, topk_group=topk_group, norm_w=True)
    ids, w = ids.cpu().numpy(), w.cpu().numpy()
    assert np.isfinite(w).all()
    assert all(len(set(r)) == k and (r >= 0).all() and (r < E).all() for r in ids)
    assert (w[:2] == 0).all() and ids[2, 0] == 17 and (w[2, 1:] == 0).all()


def test_agrees_with_topk_softmax(pkg, cuda):
    for norm in (False, True):
        lg = torch.from_numpy(zipf_logits(50, 128, seed=2)).to(cuda)
        i0, w0 = pkg.moe_cache.topk_softmax(lg, 8, norm_w=norm)
        i1, w1 = pkg.route_experts(lg, 8, norm_w=norm)
        assert torch.equal(i0, i1)
        torch.testing.assert_close(w0, w1, rtol=2 * RTOL, atol=0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_strided_and_offset_rows(pkg, cuda, dtype):
    wide = torch.from_numpy(zipf_logits(21, 83, seed=5)).to(cuda).to(dtype)
    view = wide[:, 3:67]
    ids, w = pkg.route_experts(view, 4, score="sigmoid", norm_w=True)
    i2, w2 = pkg.route_experts(view.contiguous(), 4, score="sigmoid", norm_w=True)
    assert torch.equal(ids, i2) and torch.equal(w, w2)


def test_no_tokens_and_given_outputs(pkg, cuda):
    ids, w = pkg.route_experts(torch.empty((0, 16), device=cuda), 2)
    assert ids.shape == (0, 2) and w.shape == (0, 2)
    lg = torch.randn((4, 16), device=cuda)
    ids = torch.full((4, 2), -5, dtype=torch.int32, device=cuda)
    w = torch.empty((4, 2), device=cuda)
    r = pkg.Router(2, norm_w=True)
    a, b = r(lg, ids=ids, weights=w)
    assert a is ids and b is w and (ids >= 0).all()
    for bad in (dict(ids=ids[:, :1]), dict(ids=ids.long()), dict(weights=w[:3]), dict(weights=w.t().contiguous().t())):
        with pytest.raises(pkg.MoeError):
            r(lg, **bad)
    for bad in (lg.t(), lg[None], lg.double(), lg[:, ::2]):
        with pytest.raises(pkg.MoeError):
            r(bad)
    with pytest.raises(pkg.MoeError):
        pkg.route_experts(lg, 17)
    with pytest.raises(pkg.MoeError):
        pkg.route_experts(lg, 2, bias=torch.zeros(15, device=cuda))


def test_capture_and_side_stream(pkg, cuda):
    lg = torch.randn((6, 64), device=cuda)
    b = torch.randn(64, device=cuda)
    r = pkg.Router(4, "sigmoid", bias=b, n_group=4, topk_group=2, norm_w=True)
    r(lg)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ids, w = r(lg)
    lg.copy_(torch.randn((6, 64), device=cuda))
    g.replay()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    i2, w2 = r(lg, stream=s)
    i3, w3 = r(lg, stream=s.cuda_stream)
    s.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(ids, i2) and torch.equal(w, w2) and torch.equal(ids, i3) and torch.equal(w, w3)
