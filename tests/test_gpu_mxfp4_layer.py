"""A whole layer of MXFP4 experts (router, gate/up with the GLU, down, shared
expert, combine), stage by stage on the GPU's own inputs of each stage: a
near-tie of the requantised h could otherwise move a code. And MoELayer's
GGML-format experts behind a Router."""
import numpy as np
import pytest
import torch

import mx_ref as R
from moe_data import zipf_logits

pytestmark = pytest.mark.gpu


def _blocks(rng, *shape):
    return R.to_blocks(*R.quantize_plane(0.05 * rng.normal(size=shape)))


def _layer(pkg, cuda, rng, H, F, E, k, shared=0, biases=False, op=0, **kw):
    W = {"gate": _blocks(rng, E, F, H), "up": _blocks(rng, E, F, H), "down": _blocks(rng, E, H, F)}
    if shared:
        W.update(shared_gate=_blocks(rng, shared, H), shared_up=_blocks(rng, shared, H), shared_down=_blocks(rng, H, shared))
    b = {r: 0.1 * rng.normal(size=(E, H if r == "down" else F)).astype(np.float32) for r in ("gate", "up", "down")} if biases else {}
    t = {r: pkg.moe_cache.MXFP4 for r in ("gate", "up", "down")}
    L = pkg.MoELayer(H, F, E, k, t, shared=bool(shared), weights=W, glu_op=op, device=cuda,
                     biases={r: torch.from_numpy(v).to(cuda) for r, v in b.items()}, **kw)
    assert isinstance(L, pkg.MXFP4Layer)
    return L, W, b


def _check(L, W, b, x, logits, out, op, planes, route):
    ids, w, h, y = (a.cpu().numpy() for a in L.intermediates(x.shape[0]))
    rid, rw = R.route(logits, L.k, **route)
    np.testing.assert_array_equal(ids, rid)
    np.testing.assert_allclose(w, rw, rtol=5e-6, atol=1e-37)
    u, mu = R.product(W["up"], x, ids, planes, b.get("up"))
    g, mg = R.product(W["gate"], x, ids, planes, b.get("gate"))
    du, dg = R.product_tol(mu, L.H, planes), R.product_tol(mg, L.H, planes)
    tol = (1.13 * np.abs(u) + 8.5) * dg + (np.abs(g) + 1) * du + 3e-6 * (np.abs(g) + 1) * (np.abs(u) + 1)
    assert (np.abs(h - R.glu(op, g, u)) <= tol).all()
    ref, mag = R.product(W["down"], h, ids, planes, b.get("down"))
    assert (np.abs(y - ref) <= R.product_tol(mag, L.F, planes)).all()
    want = (w[..., None].astype(np.float64) * y).sum(1)
    bound = (np.abs(w[..., None]) * np.abs(y)).sum(1) * (L.k + 1) * 2.0 ** -23
    if not L.shared:
        assert (np.abs(out - want) <= bound).all()
        return
    z = np.zeros((x.shape[0], 1), np.int32)
    su, msu = R.product(W["shared_up"][None], x, z, planes)
    sg, msg = R.product(W["shared_gate"][None], x, z, planes)
    hs = R.glu(op, sg, su)[:, 0]
    got = out - want                                       # the shared expert's part, at most a code of h apart
    ref = R.product(W["shared_down"][None], hs, z, planes)[0][:, 0]
    assert np.linalg.norm(got - ref) <= 2e-3 * np.linalg.norm(ref) + np.linalg.norm(bound)


@pytest.mark.parametrize("n", [1, 2, 9, 40, 260])
@pytest.mark.parametrize("planes", [1, 2])
def test_layer_with_groups_bias_and_shared(pkg, cuda, n, planes):
    rng = np.random.default_rng(n)
    H, F, E, k = 320, 192, 16, 4
    bias = 0.1 * rng.normal(size=E).astype(np.float32)
    route = dict(score="sigmoid", bias=bias, n_group=4, topk_group=2, group_score="top2", norm_w=True, scale=2.5)
    r = pkg.Router(k, **{**route, "bias": torch.from_numpy(bias).to(cuda)})
    L, W, b = _layer(pkg, cuda, rng, H, F, E, k, shared=160, router=r, planes=planes)
    x = rng.normal(size=(n, H)).astype(np.float32)
    lg = zipf_logits(n, E, seed=n)
    xt, lt = torch.from_numpy(x).to(cuda), torch.from_numpy(lg).to(cuda)
    out = (L.decode if n <= 8 else L.prefill)(xt, lt).cpu().numpy()
    assert pkg.moe_cache.device_error() == 0
    _check(L, W, b, x, lg, out, 0, planes, route)


@pytest.mark.parametrize("n", [1, 5, 70])
def test_layer_with_biases_and_clamped_glu(pkg, cuda, n):
    rng = np.random.default_rng(n + 50)
    H, F, E, k = 288, 352, 12, 3
    route = dict(score="softmax_topk")
    L, W, b = _layer(pkg, cuda, rng, H, F, E, k, biases=True, op=2, router=pkg.Router(k, "softmax_topk"))
    x = torch.from_numpy(rng.normal(size=(n, H)).astype(np.float32)).to(cuda).bfloat16()
    lg = torch.from_numpy(zipf_logits(n, E, seed=n)).to(cuda).bfloat16()
    out = L.decode(x, lg).cpu().numpy()
    _check(L, W, b, x.float().cpu().numpy(), lg.float().cpu().numpy(), out, 2, 2, route)


def test_default_router_trace_capture_and_given_out(pkg, cuda, tmp_path):
    rng = np.random.default_rng(3)
    L, W, b = _layer(pkg, cuda, rng, 128, 64, 8, 2)
    x, lg = torch.randn((3, 128), device=cuda), torch.from_numpy(zipf_logits(3, 8, seed=1)).to(cuda)
    out = L.decode(x, lg)
    i, w = pkg.moe_cache.topk_softmax(lg, 2)
    assert torch.equal(L.routing_of(3)[0], i)
    from importlib import import_module
    seed = import_module("a6000-custom-kernels_b200.seed")
    path = tmp_path / "t.bin"
    tw = seed.TraceWriter(str(path))
    assert torch.equal(L.decode(x, lg, trace=tw), out)
    given = torch.empty((3, 128), device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    assert L.decode(x, lg, out=given, stream=s) is given
    torch.cuda.synchronize()
    assert torch.equal(given, out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.decode(x, lg, out=given)
    given.zero_()
    g.replay()
    assert torch.equal(given, out)
    assert L.decode(x[:0], lg[:0]).shape == (0, 128)
    assert L.weight_bytes_per_token() == 2 * (3 * 8704) and not L.fused(1)
    with pytest.raises(pkg.MoeError):
        L.decode(x[:, :64], lg)
    with pytest.raises(pkg.MoeError):
        L.decode(x, lg, out=given[:, :64])


def test_random_weights_layer_runs(pkg, cuda):
    L = pkg.MoELayer(256, 128, 8, 2, {r: pkg.moe_cache.MXFP4 for r in ("gate", "up", "down")}, device=cuda, seed=4)
    out = L.prefill(torch.randn((20, 256), device=cuda), torch.randn((20, 8), device=cuda))
    assert torch.isfinite(out).all() and out.abs().max() > 0


@pytest.mark.parametrize("t", [10, 2])          # Q2_K, Q4_0
@pytest.mark.parametrize("n", [1, 5, 40])
def test_ggml_layer_behind_a_router(pkg, cuda, t, n):
    """MoELayer(router=...): the default router's result with a softmax Router (same picks, weights to their
    rounding), and the weighted sum of its experts for another one."""
    pkg.moe_cache.configure(enabled=True)
    try:
        H, F, E, k = 512, 256, 16, 4
        types = {r: t for r in ("gate", "up", "down")}
        base = pkg.MoELayer(H, F, E, k, types, device=cuda, seed=2)
        x = torch.randn((n, H), device=cuda)
        lg = torch.from_numpy(zipf_logits(n, E, seed=n)).to(cuda)
        soft = pkg.MoELayer(H, F, E, k, types, device=cuda, seed=2, router=pkg.Router(k))
        a, b = base.prefill(x, lg), soft.prefill(x, lg)
        assert (a - b).abs().max() <= 2e-5 * a.abs().max()
        assert torch.equal(soft.decode(x, lg), b)
        r = pkg.Router(k, "sigmoid", bias=torch.randn(E, device=cuda), n_group=4, topk_group=2, norm_w=True, scale=2.0)
        other = pkg.MoELayer(H, F, E, k, types, device=cuda, seed=2, router=r, shared=False)
        got = other.prefill(x, lg)
        ids, w = r(lg)
        y = other._ws[("routed", n)][1]
        want = (w.double()[..., None] * y.double()).sum(1)
        assert (got - want).abs().max() <= 1e-6 * (w[..., None] * y).abs().sum(1).max()
        each = pkg.MoELayer(H, F, E, 1, types, device=cuda, seed=2, shared=False, router=pkg.Router(1, "softmax_topk"))
        one = each.prefill(x, torch.nn.functional.one_hot(ids[:, 0].long(), E).float())
        assert (one - y[:, 0]).abs().max() <= 1e-6 * y.abs().max()
    finally:
        pkg.moe_cache.reset()


def test_trace_names_and_streams(pkg, cuda, tmp_path):
    """The trace has the layer's name and the picks of the stream that the call ran on; a router's bias written
    in place takes effect."""
    from importlib import import_module
    seed = import_module("a6000-custom-kernels_b200.seed")
    bias = torch.zeros(8, device=cuda)
    t = {r: pkg.moe_cache.MXFP4 for r in ("gate", "up", "down")}
    L = pkg.MoELayer(64, 64, 8, 2, t, False, device=cuda, name="blk.7", router=pkg.Router(2, "sigmoid", bias=bias))
    x, lg = torch.randn((4, 64), device=cuda), torch.randn((4, 8), device=cuda)
    path = tmp_path / "t.bin"
    with seed.TraceWriter(str(path)) as tw:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        L.decode(x, lg, stream=s, trace=tw)
        torch.cuda.synchronize()
        bias[5] = 10.0
        L.decode(x, lg, trace=tw)
    rec = list(seed.read_trace(str(path)))
    assert [r[0] for r in rec] == 2 * [f"blk.7.ffn_{r}_exps.weight" for r in ("gate", "up", "down")]
    ids = pkg.route_experts(lg, 2, "sigmoid")[0].cpu().numpy()
    np.testing.assert_array_equal(np.asarray(rec[0][-1]).reshape(4, 2), ids)
    assert (np.asarray(rec[3][-1]).reshape(4, 2)[:, 0] == 5).all()


def test_router_layer_refusals(pkg, cuda):
    pkg.moe_cache.configure(enabled=True)
    try:
        types = {r: pkg.moe_cache.Q4_0 for r in ("gate", "up", "down")}
        L = pkg.MoELayer(256, 128, 8, 2, types, False, device=cuda, router=pkg.Router(2, "sigmoid"))
        x, lg = torch.randn((3, 256), device=cuda), torch.randn((3, 8), device=cuda)
        for kw in (dict(x=x.half()), dict(x=x[:, :128]), dict(x=x.cpu()), dict(logits=lg.cpu()), dict(logits=lg[:2]),
                   dict(out=torch.empty((3, 255), device=cuda)), dict(out=torch.empty((3, 256), device=cuda).half())):
            with pytest.raises(pkg.MoeError):
                L.decode(**{**dict(x=x, logits=lg), **kw})
        assert torch.isfinite(L.decode(x, lg)).all()
    finally:
        pkg.moe_cache.reset()


def test_more_tokens_than_a_grid_has_rows(pkg, cuda):
    t = {r: pkg.moe_cache.MXFP4 for r in ("gate", "up", "down")}
    L = pkg.MoELayer(32, 32, 2, 1, t, device=cuda, planes=1)
    n = 65535 + 70
    x, lg = torch.randn((n, 32), device=cuda), torch.randn((n, 2), device=cuda)
    out = L.prefill(x, lg)
    part = L.prefill(x[-100:], lg[-100:])
    assert torch.equal(out[-100:], part) and torch.equal(out[:100], L.prefill(x[:100], lg[:100]))
