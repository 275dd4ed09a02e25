"""Calls of the MXFP4 operators that the documentation allows, off the main
path: short last runs of a row, waits that give up, streams, graphs, given
planes. Values against the 64-bit reference (mx_ref)."""
import numpy as np
import pytest
import torch

import mx_ref as R

pytestmark = pytest.mark.gpu


def _experts(rng, E, rows, K):
    return R.to_blocks(*R.quantize_plane(0.02 * rng.normal(size=(E, rows, K))))


def _weights(pkg, cuda, blocks, K):
    return pkg.MXFP4Weights(torch.from_numpy(blocks).to(cuda), K, blocks.shape[1])


def _ids(rng, n, k, E):
    return np.argsort(rng.normal(size=(n, E)), axis=1)[:, :k].astype(np.int32)


@pytest.mark.parametrize("planes", [1, 2])
@pytest.mark.parametrize("n,K", [(5500, 352), (4097, 608), (2400, 896)])   # 3, 5 and 7 K tiles
def test_long_prompt_with_an_odd_number_of_tiles(pkg, cuda, n, K, planes):
    """Rows whose tiles the halves of a warp share unevenly: one of them is at its row's last, single tile."""
    rng = np.random.default_rng(K)
    E, rows = 3, 40
    W = _experts(rng, E, rows, K)
    x = rng.normal(size=(n, K)).astype(np.float32)
    ids = rng.integers(0, E, size=(n, 1)).astype(np.int32)
    y = pkg.mxfp4_mul_mat_id(_weights(pkg, cuda, W, K), torch.from_numpy(x).to(cuda), torch.from_numpy(ids).to(cuda),
                             planes=planes).cpu().numpy()
    ref, mag = R.product(W, x, ids, planes)
    assert pkg.moe_cache.device_error() == 0
    assert (np.abs(y - ref) <= R.product_tol(mag, K, planes)).all()


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("n,k,E,K,rows", [
    (1, 4, 8, 2048, 256),      # K shared by a cluster
    (8, 8, 64, 768, 1024),     # more tiles than CTAs
    (40, 2, 8, 1024, 256),     # grouped: 16 columns,
    (60, 4, 8, 512, 256),      # 64,
    (300, 4, 8, 512, 256),     # and the widest
])
def test_whichever_warp_gives_up(pkg, cuda, n, k, E, K, rows, glu):
    """Wait limits from nothing to a little less than the kernel's time, so that the copies', the MMAs' and the
    epilogue's waits are the ones that run out: what is in flight ends before the CTA's memory goes, and the next call
    is right."""
    mc = pkg.moe_cache
    rng = np.random.default_rng(n)
    w = _weights(pkg, cuda, _experts(rng, E, rows, K), K)
    x = torch.from_numpy(rng.normal(size=(n, K)).astype(np.float32)).to(cuda)
    ids = torch.from_numpy(_ids(rng, n, k, E)).to(cuda)
    kw = dict(gate=w) if glu else {}
    good = pkg.mxfp4_mul_mat_id(w, x, ids, **kw)
    assert mc.device_error() == 0
    for limit in (1, 250, 500, 1000, 1500, 2000, 3000, 5000, 10000, 19000):
        try:
            mc.set_wait_limits(kernel_wait_ns=limit)
            pkg.mxfp4_mul_mat_id(w, x, ids, **kw)
            code = mc.device_error()
        finally:
            mc.set_wait_limits()
        assert code in (0, mc.DERR_TIMEOUT_FULL)
        assert torch.equal(pkg.mxfp4_mul_mat_id(w, x, ids, **kw), good)
        assert mc.device_error() == 0


def test_a_graph_outlives_the_caches_reset(pkg, cuda):
    """moe_b200_reset frees the cache's state; a captured product still reports a bad id, and a product captured
    right after it needs no eager call first."""
    mc = pkg.moe_cache
    rng = np.random.default_rng(1)
    w = _weights(pkg, cuda, _experts(rng, 4, 130, 96), 96)
    x = torch.from_numpy(rng.normal(size=(6, 96)).astype(np.float32)).to(cuda)
    ids = torch.zeros((6, 2), dtype=torch.int32, device=cuda)
    mc.configure(enabled=True)
    want = pkg.mxfp4_mul_mat_id(w, x, ids)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = pkg.mxfp4_mul_mat_id(w, x, ids)
    mc.reset()
    g.replay()
    assert mc.device_error() == 0 and torch.equal(y, want)
    ids[3, 1] = 9
    g.replay()
    assert mc.device_error() == mc.DERR_BAD_ID and mc.device_error() == 0
    ids[3, 1] = 0
    mc.reset()
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        y2 = pkg.mxfp4_mul_mat_id(w, x, ids)
    g2.replay()
    assert mc.device_error() == 0 and torch.equal(y2, want)


@pytest.mark.parametrize("n", [1, 2, 3])
def test_read_back_without_a_word_on_planes(pkg, cuda, n):
    """What quantize_mxfp4 returned is read back as it was made, whatever its first dimension; blocks from
    elsewhere whose first dimension could count planes are refused."""
    x = torch.randn((n, 5, 64), device=cuda)
    for planes in (1, 2):
        q = pkg.quantize_mxfp4(x, planes=planes)
        back = pkg.dequantize_mxfp4(q, 64)
        assert back.shape == x.shape and torch.equal(back, pkg.dequantize_mxfp4(q, 64, planes=planes))
        rows = pkg.quantize_mxfp4(x[:, 0], planes=planes)
        assert torch.equal(pkg.dequantize_mxfp4(rows, 64), back[:, 0])
        foreign = q.clone()
        if foreign.shape[0] == 2:
            with pytest.raises(pkg.MoeError, match="planes"):
                pkg.dequantize_mxfp4(foreign, 64)
        else:
            assert torch.equal(pkg.dequantize_mxfp4(foreign, 64), back)
        assert torch.equal(pkg.dequantize_mxfp4(foreign, 64, planes=planes), back)
    buf = torch.empty((2, 5, 34), dtype=torch.uint8, device=cuda)
    one, two = torch.randn((2, 5, 64), device=cuda), torch.randn((5, 64), device=cuda)
    assert pkg.dequantize_mxfp4(pkg.quantize_mxfp4(one, out=buf), 64).shape == (2, 5, 64)      # one buffer, both ways
    assert pkg.dequantize_mxfp4(pkg.quantize_mxfp4(two, planes=2, out=buf), 64).shape == (5, 64)
    buf.copy_(pkg.quantize_mxfp4(one))                      # written by something else: says nothing any more
    with pytest.raises(pkg.MoeError, match="planes"):
        pkg.dequantize_mxfp4(buf, 64)
    pkg.quantize_mxfp4(two, planes=2, out=buf)
    pkg.quantize_mxfp4(one, out=buf.view(2, 5, 34))         # so says a view of it
    with pytest.raises(pkg.MoeError, match="planes"):
        pkg.dequantize_mxfp4(buf, 64)
    with torch.inference_mode():
        assert pkg.dequantize_mxfp4(pkg.quantize_mxfp4(one), 64).shape == (2, 5, 64)
        assert pkg.dequantize_mxfp4(pkg.quantize_mxfp4(two, planes=2), 64).shape == (5, 64)


def _behind_a_busy_stream(call, *inputs):
    """call(stream, temporaries) on a stream that is busy; the temporaries go and their memory is taken again and
    overwritten before the stream comes to the call."""
    s = torch.cuda.Stream()
    tmp = [t.clone() for t in inputs]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(60_000_000)
    out = call(s, tmp)
    del tmp
    junk = [torch.zeros_like(t) for t in inputs]
    torch.cuda.synchronize()
    assert all((j == 0).all() for j in junk)
    return out


def test_temporaries_on_another_stream(pkg, cuda):
    """Inputs that the caller drops right behind a call on another stream keep their memory until it has run."""
    rng = np.random.default_rng(2)
    n, K, E, k = 2048, 1024, 8, 2
    w = _weights(pkg, cuda, _experts(rng, E, 64, K), K)
    x = torch.randn((n, K), device=cuda)
    ids = torch.from_numpy(_ids(rng, n, k, E)).to(cuda)
    bias = torch.randn((E, 64), device=cuda)
    lg = torch.randn((n, 256), device=cuda)
    rb = torch.randn(256, device=cuda)
    blocks = pkg.quantize_mxfp4(x)
    wide = torch.from_numpy(_experts(rng, 2, 512, K)).to(cuda)
    layer = pkg.MoELayer(K, 64, E, k, {r: pkg.moe_cache.MXFP4 for r in ("gate", "up", "down")}, device=cuda)
    l8 = torch.randn((n, E), device=cuda)
    xs, i1 = torch.randn((4, K), device=cuda), torch.zeros((4, 1), dtype=torch.int32, device=cuda)
    for call, inputs in (
            (lambda s, t: pkg.quantize_mxfp4(t[0], stream=s), (x,)),
            (lambda s, t: pkg.dequantize_mxfp4(t[0], K, stream=s), (blocks,)),
            (lambda s, t: pkg.mxfp4_mul_mat_id(w, t[0], t[1], bias=t[2], stream=s), (x, ids, bias)),
            (lambda s, t: pkg.mxfp4_mul_mat_id(w, t[0], t[1], gate=w, bias=t[2], gate_bias=t[2], stream=s), (x, ids, bias)),
            (lambda s, t: pkg.route_experts(t[0], 4, bias=t[1], stream=s), (lg, rb)),
            (lambda s, t: pkg.MXFP4Weights(t[0], K, 512, stream=s).data, (wide,)),
            (lambda s, t: layer.decode(t[0], t[1], stream=s), (x, l8))):
        here = call(None, inputs)
        got = _behind_a_busy_stream(call, *inputs)
        for a, b in zip(got, here) if isinstance(here, tuple) else ((got, here),):
            assert torch.equal(a, b)
    # matrices that go right behind the call that uses them
    packed = lambda: pkg.MXFP4Weights(wide, K, 512)   # noqa: E731
    here = pkg.mxfp4_mul_mat_id(packed(), xs, i1)
    s = torch.cuda.Stream()
    m = packed()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(60_000_000)
    y = pkg.mxfp4_mul_mat_id(m, xs, i1, stream=s)
    size = m.data.numel()
    del m
    junk = torch.zeros(size, dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()
    assert torch.equal(y, here) and not junk.any()


def test_captured_with_a_forked_stream(pkg, cuda):
    """A capture that forks: calls on another stream, on temporaries of the capturing one that go right behind them,
    joined again; then eager calls, and the replays are right."""
    rng = np.random.default_rng(6)
    n, K, E, k = 300, 512, 8, 2
    w = _weights(pkg, cuda, _experts(rng, E, 200, K), K)
    layer = pkg.MoELayer(K, 64, E, k, {r: pkg.moe_cache.MXFP4 for r in ("gate", "up", "down")}, device=cuda)
    x, lg = torch.randn((n, K), device=cuda), torch.randn((n, E), device=cuda)
    ids = torch.from_numpy(_ids(rng, n, k, E)).to(cuda)

    def calls(x, lg, s=None):
        return (pkg.mxfp4_mul_mat_id(w, x, ids, gate=w, stream=s), layer.decode(x, lg, stream=s),
                pkg.dequantize_mxfp4(pkg.quantize_mxfp4(x, planes=2, stream=s), K, stream=s))
    want = calls(x * 2, lg * 2)
    torch.cuda.synchronize()
    fork = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, b = x * 2, lg * 2
        fork.wait_stream(torch.cuda.current_stream())
        out = calls(a, b, fork)
        del a, b
        junk = [torch.zeros((n, K), device=cuda) for _ in range(4)]
        torch.cuda.current_stream().wait_stream(fork)
    for _ in range(3):
        for o in out:
            o.zero_()
        calls(torch.randn((n, K), device=cuda), lg)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert not any(j.any() for j in junk)
