"""The MXFP4 quantiser, its read-back and the experts' product against the
64-bit reference (mx_ref). Quantised bytes and read-back values are equal
exactly: every step of theirs is a comparison or exact. Products: mx_ref.product_tol."""
import numpy as np
import pytest
import torch

import mx_ref as R

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rows(rng, n, K, dtype, cuda):
    x = rng.normal(size=(n, K)) * np.exp2(rng.integers(-6, 7, size=(n, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(cuda).to(dtype)


def _edge_rows():
    """Blocks that decide something: zeros, one value, ties, powers of two, saturation, tiny and huge numbers."""
    x = np.zeros((14, 64), np.float64)
    x[1, 3] = 1.0
    x[2, :32] = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4) * np.tile([1, -1], 16)   # every tie
    x[3] = 7.999 * np.where(np.arange(64) % 2, 1, -1)        # all saturate
    x[4, 0], x[4, 40] = 2.0 ** -126, 2.0 ** -140             # the smallest scales
    x[5, :] = 2.0 ** -149
    x[6, 1], x[6, 33] = 3e38, -3.4e38
    x[7, :] = -0.0
    x[8, :32] = np.linspace(-8, 8, 32)
    x[9, 7], x[9, 8] = 4.0, 3.9999998
    x[10, 31], x[10, 32] = 65504.0, 6e-8
    x[11, 5], x[12, 37], x[13, 0] = np.inf, -np.inf, np.nan
    return x


@pytest.mark.parametrize("planes", [1, 2])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_edges(pkg, cuda, dtype, planes):
    x = torch.from_numpy(_edge_rows().astype(np.float32)).to(cuda).to(dtype)
    got = pkg.quantize_mxfp4(x, planes=planes).cpu().numpy().reshape(planes, 14, -1)
    with np.errstate(invalid="ignore"):
        want = R.quantize(x.float().cpu().numpy(), planes)
    for p in range(planes):
        np.testing.assert_array_equal(got[p], want[p])


@pytest.mark.parametrize("planes", [1, 2])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,K,wide", [(1, 32, 0), (3, 96, 0), (1, 8192, 0), (33, 160, 5), (257, 1440, 48), (7, 64, 4), (130, 2048, 0)])
def test_quantize_and_read_back(pkg, cuda, n, K, wide, dtype, planes):
    rng = np.random.default_rng(n + K)
    x = _rows(rng, n, K + wide, dtype, cuda)[:, wide - wide // 2: K + wide - wide // 2]
    q = pkg.quantize_mxfp4(x, planes=planes)
    want = R.quantize(x.float().cpu().numpy(), planes)
    got = q.cpu().numpy().reshape(planes, n, -1)
    for p in range(planes):
        np.testing.assert_array_equal(got[p], want[p])
    val = sum(R.from_blocks(b, K) for b in want)
    for out in DTYPES:
        back = pkg.dequantize_mxfp4(q, K, planes=planes, dtype=out)
        ref = torch.from_numpy(val).to(torch.float32).to(out)          # exact in f32, rounded once
        assert torch.equal(back.cpu(), ref)


def test_read_back_of_any_bytes(pkg, cuda):
    """Every scale byte and code, NaN scales among them, and planes that are not of one number."""
    rng = np.random.default_rng(4)
    b = rng.integers(0, 256, size=(2, 256, 34), dtype=np.uint8)
    b[:, :, 0] = np.arange(256)
    b[1, :, 17] = np.minimum(b[0, :, 17], 254)
    got = pkg.dequantize_mxfp4(torch.from_numpy(b[0]).to(cuda), 64).cpu().numpy()
    np.testing.assert_array_equal(got, R.from_blocks(b[0], 64).astype(np.float32))
    two = pkg.dequantize_mxfp4(torch.from_numpy(b).to(cuda), 64, planes=2).cpu().numpy()
    with np.errstate(over="ignore", invalid="ignore"):
        ref = R.from_blocks(b[0], 64).astype(np.float32) + R.from_blocks(b[1], 64).astype(np.float32)
    np.testing.assert_array_equal(two, ref)


@pytest.mark.parametrize("offset", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("n", [5, 64, 300])
def test_blocks_at_any_alignment(pkg, cuda, n, offset):
    """Blocks inside a larger byte buffer; what lies around them stays."""
    rng = np.random.default_rng(n)
    x = _rows(rng, n, 96, torch.float32, cuda)
    nbytes = 2 * n * 51
    buf = torch.full((nbytes + 64,), 77, dtype=torch.uint8, device=cuda)
    out = buf[offset: offset + nbytes].view(2, n, 51)
    pkg.quantize_mxfp4(x, planes=2, out=out)
    ref = pkg.quantize_mxfp4(x, planes=2)
    assert torch.equal(out, ref)
    assert (buf[:offset] == 77).all() and (buf[offset + nbytes:] == 77).all()
    vals = torch.full((n + 2, 100), 5.0, device=cuda)
    pkg.dequantize_mxfp4(out, 96, out=vals[1: n + 1, 1:97])
    assert torch.equal(vals[1: n + 1, 1:97], pkg.dequantize_mxfp4(ref, 96))
    assert (vals[0] == 5).all() and (vals[-1] == 5).all() and (vals[:, 0] == 5).all() and (vals[:, 97:] == 5).all()


def test_quantize_shapes_and_refusals(pkg, cuda):
    x = torch.randn((2, 3, 64), device=cuda)
    assert pkg.quantize_mxfp4(x).shape == (2, 3, 34)
    q = pkg.quantize_mxfp4(x, planes=2)
    assert q.shape == (2, 2, 3, 34) and pkg.dequantize_mxfp4(q, 64, planes=2).shape == (2, 3, 64)
    assert pkg.quantize_mxfp4(x[:0]).shape == (0, 3, 34) and pkg.dequantize_mxfp4(q[:, :0], 64, planes=2).shape == (0, 3, 64)
    for bad in (x[..., :48], x.transpose(0, 1), x[..., ::2], x[:, :, 0], x.double(), x[:1].expand(2, 3, 64)):
        with pytest.raises(pkg.MoeError):
            pkg.quantize_mxfp4(bad)
    with pytest.raises(pkg.MoeError):
        pkg.quantize_mxfp4(x, planes=3)
    with pytest.raises(pkg.MoeError):
        pkg.quantize_mxfp4(x, out=torch.empty((2, 3, 33), dtype=torch.uint8, device=cuda))
    for kw in (dict(K=32), dict(K=64, dtype=torch.float64), dict(K=64, planes=3)):
        with pytest.raises(pkg.MoeError):
            pkg.dequantize_mxfp4(q, **kw)


# ---- the product ------------------------------------------------------------------

def _experts(rng, E, rows, K):
    return R.to_blocks(*R.quantize_plane(0.02 * rng.normal(size=(E, rows, K)) * np.exp2(rng.integers(-2, 3, size=(E, rows, 1)))))


def _weights(pkg, cuda, blocks, K):
    return pkg.MXFP4Weights(torch.from_numpy(blocks).to(cuda), K, blocks.shape[1])


def _ids(rng, n, k, E, skew=1.1):
    lg = -skew * np.log(rng.permutation(E) + 1.0) + rng.normal(size=(n, E))
    return np.argsort(-lg, axis=1, kind="stable")[:, :k].astype(np.int32)


def _run(pkg, cuda, W, x, ids, K, planes, dtype=torch.float32, bias=None, dst=None):
    w = _weights(pkg, cuda, W, K)
    xt = torch.from_numpy(x.astype(np.float32)).to(cuda).to(dtype)
    b = None if bias is None else torch.from_numpy(bias.astype(np.float32)).to(cuda)
    y = pkg.mxfp4_mul_mat_id(w, xt, torch.from_numpy(ids).to(cuda), bias=b, planes=planes, dst=dst)
    torch.cuda.synchronize()
    return y.cpu().numpy(), xt.float().cpu().numpy()


@pytest.mark.parametrize("planes", [1, 2])
@pytest.mark.parametrize("n,k,E,K,rows,per_pick,bias,dtype", [
    (1, 1, 1, 32, 1, False, False, torch.float32),        # one block, one row
    (1, 4, 8, 96, 129, False, True, torch.float32),       # padded K and rows
    (1, 8, 16, 2048, 256, False, False, torch.bfloat16),  # one token, K shared by a cluster
    (2, 3, 4, 1440, 100, True, True, torch.float16),
    (8, 8, 16, 768, 300, True, False, torch.float32),     # 64 entries: the last direct size
    (13, 5, 16, 256, 128, False, True, torch.float32),    # 65: grouped
    (40, 1, 2, 512, 200, False, False, torch.float32),    # one pick each: more than a chunk of one expert
    (16, 4, 4, 160, 384, False, False, torch.bfloat16),   # every token picks every expert
    (1, 1, 2, 24544, 128, False, True, torch.float16),    # a ring that is used several times over
    (16, 4, 64, 8224, 128, False, True, torch.float16),   # and by several chunks
    (16, 2, 2, 2048, 128, False, False, torch.float32),   # more rows to a chunk than the product quantises
    (17, 3, 8, 416, 130, False, False, torch.float32),    # some experts in several chunks
    (64, 1, 1, 352, 128, False, True, torch.bfloat16),    # one expert, four full chunks
    (100, 4, 8, 384, 250, True, True, torch.float32),     # chunks of 64
    (300, 4, 4, 256, 256, False, False, torch.float32),   # the widest chunks, an even number of row tiles
    (500, 2, 3, 640, 390, True, True, torch.bfloat16),    # and an odd one
    (77, 6, 200, 128, 64, False, False, torch.float32),   # more experts than entries of most
    (1100, 8, 16, 64, 48, False, False, torch.float32),   # many entries
])
def test_product(pkg, cuda, n, k, E, K, rows, per_pick, bias, dtype, planes):
    rng = np.random.default_rng(n * 7 + K)
    W = _experts(rng, E, rows, K)
    x = rng.normal(size=(n, k, K) if per_pick else (n, K)) * np.exp2(rng.integers(-3, 4, size=(n,) + (1,) * (2 if per_pick else 1)))
    ids = _ids(rng, n, k, E)
    b = 0.1 * rng.normal(size=(E, rows)).astype(np.float32) if bias else None
    y, xv = _run(pkg, cuda, W, x, ids, K, planes, dtype, b)
    ref, mag = R.product(W, xv, ids, planes, b)
    assert pkg.moe_cache.device_error() == 0
    assert (np.abs(y - ref) <= R.product_tol(mag, K, planes)).all()


@pytest.mark.parametrize("op", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("n,k,E,K,rows,planes,bias", [
    (1, 4, 8, 1024, 200, 2, True), (6, 2, 4, 96, 130, 1, False), (30, 4, 8, 320, 128, 2, True), (90, 4, 6, 256, 260, 1, True),
    (260, 4, 5, 192, 200, 2, False), (9, 1, 3, 512, 64, 1, True),
])
def test_product_with_glu(pkg, cuda, n, k, E, K, rows, planes, bias, op):
    """dst = GLU(gate . x + gate_bias, w . x + bias). The GLU's own error: its sums' errors times its slopes --
    every op here moves by at most 1.13 |u| + 8.5 per unit of g (geglu, the steepest, 1.13; swiglu 1.1; the
    clamped ones less; the product |u|) and by |G(g)| + 1 per unit of u -- plus 3e-6 of the value's factors for
    exp, tanh and the quotients in 32 bits."""
    rng = np.random.default_rng(n + 10 * op)
    U, G = _experts(rng, E, rows, K), _experts(rng, E, rows, K)
    x = rng.normal(size=(n, K)).astype(np.float32)
    ids = _ids(rng, n, k, E)
    bu, bg = (rng.normal(size=(E, rows)).astype(np.float32) for _ in range(2)) if bias else (None, None)
    limit = 1.25
    t = lambda a: None if a is None else torch.from_numpy(a).to(cuda)   # noqa: E731
    y = pkg.mxfp4_mul_mat_id(_weights(pkg, cuda, U, K), t(x), t(ids), gate=_weights(pkg, cuda, G, K), bias=t(bu), gate_bias=t(bg),
                             glu_op=op, glu_limit=limit, planes=planes).cpu().numpy()
    u, mu = R.product(U, x, ids, planes, bu)
    g, mg = R.product(G, x, ids, planes, bg)
    ref = R.glu(op, g, u, limit)
    du, dg = R.product_tol(mu, K, planes), R.product_tol(mg, K, planes)
    tol = (1.13 * np.abs(u) + 8.5) * dg + (np.abs(g) + 1) * du + 3e-6 * (np.abs(g) + 1) * (np.abs(u) + 1)
    assert (np.abs(y - ref) <= tol).all()


def test_same_expert_twice(pkg, cuda):
    """One expert several times among a token's picks, and one expert for everything."""
    rng = np.random.default_rng(5)
    E, K, rows = 6, 256, 140
    W = _experts(rng, E, rows, K)
    for ids in (np.array([[2, 2, 5, 2], [5, 5, 5, 5], [0, 1, 0, 1]], np.int32), np.full((90, 3), 4, np.int32),
                rng.integers(0, E, size=(45, 7)).astype(np.int32)):
        x = rng.normal(size=ids.shape + (K,))
        y, xv = _run(pkg, cuda, W, x, ids, K, 2)
        ref, mag = R.product(W, xv, ids, 2)
        assert (np.abs(y - ref) <= R.product_tol(mag, K, 2)).all()


@pytest.mark.parametrize("n", [5, 40, 400])
@pytest.mark.parametrize("glu", [False, True])
def test_skipped_and_bad_ids_leave_their_rows(pkg, cuda, n, glu):
    rng = np.random.default_rng(n)
    E, K, rows, k = 8, 128, 130, 4
    W = _experts(rng, E, rows, K)
    w = _weights(pkg, cuda, W, K)
    x = rng.normal(size=(n, K)).astype(np.float32)
    ids = _ids(rng, n, k, E)
    ids[rng.random(size=ids.shape) < 0.3] = -1
    ids[0] = -1                                  # a padded row
    xt, mark = torch.from_numpy(x).to(cuda), 123.0
    pkg.moe_cache.device_error()

    def go(i):
        dst = torch.full((n, k, rows), mark, device=cuda)
        kw = dict(gate=w, glu_op=4) if glu else {}
        pkg.mxfp4_mul_mat_id(w, xt, torch.from_numpy(i).to(cuda), dst=dst, **kw)
        return dst.cpu().numpy()
    y = go(ids)
    assert pkg.moe_cache.device_error() == 0
    ref, mag = R.product(W, x, ids, 2)
    tol = R.product_tol(mag, K, 2)
    if glu:
        ref, tol = ref * ref, 2 * np.abs(ref) * tol + tol * tol + 2.0 ** -23 * ref * ref
    out = ids < 0
    assert (y[out] == mark).all()
    assert (np.abs(y - ref)[~out] <= tol[~out]).all()
    worse = ids.copy()
    worse[n // 2, 1], worse[n - 1, 0] = E, -7
    y2 = go(worse)
    assert pkg.moe_cache.device_error() == pkg.moe_cache.DERR_BAD_ID
    out = (worse < 0) | (worse >= E)
    assert (y2[out] == mark).all() and np.array_equal(y2[~out], y[~out])
    assert (go(np.full_like(ids, -1)) == mark).all()
    assert pkg.moe_cache.device_error() == 0


@pytest.mark.parametrize("n", [3, 50, 300])
def test_nan_and_infinity_stay_in_their_row(pkg, cuda, n):
    rng = np.random.default_rng(n)
    E, K, rows, k = 4, 160, 129, 2
    W = _experts(rng, E, rows, K)
    x = rng.normal(size=(n, K)).astype(np.float32)
    ids = _ids(rng, n, k, E)
    clean, _ = _run(pkg, cuda, W, x, ids, K, 2)
    x[1, 7], x[n - 1, 150] = np.nan, -np.inf
    y, _ = _run(pkg, cuda, W, x, ids, K, 2)
    bad = np.zeros(n, bool)
    bad[[1, n - 1]] = True
    assert np.isnan(y[bad]).all() and np.array_equal(y[~bad], clean[~bad])
    W[2, 3, 17] = 255                            # a NaN scale in row 3 of expert 2
    y, _ = _run(pkg, cuda, W, x, ids, K, 2)
    hit = (ids == 2) & ~bad[:, None]
    assert np.isnan(y[..., 3][hit]).all()
    rest = np.delete(y, 3, axis=2)[~bad]
    assert np.array_equal(rest, np.delete(clean, 3, axis=2)[~bad])


def test_zero_rows_and_extreme_scales(pkg, cuda):
    rng = np.random.default_rng(9)
    K, rows, E = 128, 64, 2
    W = _experts(rng, E, rows, K)
    W[0, 0] = 0                                  # scale byte 0, zero codes
    x = rng.normal(size=(4, K))
    x[1] = 0
    x[2] *= 1e30
    x[3] *= 1e-30
    ids = np.array([[0, 1]] * 4, np.int32)
    y, xv = _run(pkg, cuda, W, x, ids, K, 2)
    ref, mag = R.product(W, xv, ids, 2)
    assert (np.abs(y - ref) <= R.product_tol(mag, K, 2)).all()
    assert (y[1] == 0).all() and (y[:, 0, 0] == 0).all()


@pytest.mark.parametrize("n", [4, 100, 400])
def test_equal_calls_equal_bits(pkg, cuda, n):
    rng = np.random.default_rng(n)
    W = _experts(rng, 8, 256, 1024)
    x = rng.normal(size=(n, 1024))
    ids = _ids(rng, n, 4, 8)
    first, _ = _run(pkg, cuda, W, x, ids, 1024, 2)
    for _ in range(3):
        assert np.array_equal(_run(pkg, cuda, W, x, ids, 1024, 2)[0], first)


def test_strides_of_x_and_ids(pkg, cuda):
    rng = np.random.default_rng(1)
    W = _experts(rng, 4, 96, 96)
    w = _weights(pkg, cuda, W, 96)
    for n in (3, 60):
        wide = torch.from_numpy(rng.normal(size=(n, 140)).astype(np.float32)).to(cuda)
        ids_wide = torch.from_numpy(np.concatenate([_ids(rng, n, 3, 4), np.full((n, 2), 99, np.int32)], 1)).to(cuda)
        for dtype in DTYPES:
            x, ids = wide.to(dtype)[:, 1:97], ids_wide[:, :3]
            assert torch.equal(pkg.mxfp4_mul_mat_id(w, x, ids), pkg.mxfp4_mul_mat_id(w, x.contiguous(), ids.contiguous()))
        xp = torch.randn((n, 3, 128), device=cuda)[..., 32:]
        assert torch.equal(pkg.mxfp4_mul_mat_id(w, xp, ids), pkg.mxfp4_mul_mat_id(w, xp.contiguous(), ids.contiguous()))


def test_no_tokens_and_refusals(pkg, cuda):
    rng = np.random.default_rng(2)
    w = _weights(pkg, cuda, _experts(rng, 4, 64, 64), 64)
    other = _weights(pkg, cuda, _experts(rng, 4, 32, 64), 64)
    assert pkg.mxfp4_mul_mat_id(w, torch.empty((0, 64), device=cuda), torch.empty((0, 2), dtype=torch.int32, device=cuda)).shape == (0, 2, 64)
    x, ids = torch.randn((3, 64), device=cuda), torch.zeros((3, 2), dtype=torch.int32, device=cuda)
    good = dict(w=w, x=x, ids=ids)
    for kw in (dict(x=x[:2]), dict(x=x[:, :32]), dict(x=x.double()), dict(x=x.cpu()), dict(ids=ids.long()), dict(ids=ids[:, 0]),
               dict(ids=ids[:1].expand(3, 2)), dict(gate=other), dict(gate_bias=torch.zeros((4, 64), device=cuda)),
               dict(bias=torch.zeros((4, 63), device=cuda)), dict(bias=torch.zeros((4, 64), device=cuda).half()), dict(planes=3),
               dict(dst=torch.empty((3, 2, 63), device=cuda)), dict(workspace=torch.empty(16, device=cuda)),
               dict(x=x.repeat(11, 1), ids=ids.repeat(11, 1), workspace=torch.empty(16, dtype=torch.uint8, device=cuda)),
               dict(x=torch.randn((3, 3, 64), device=cuda)), dict(gate=w, glu_op=7)):
        with pytest.raises(pkg.MoeError):
            pkg.mxfp4_mul_mat_id(**{**good, **kw})
    with pytest.raises(pkg.MoeError):
        pkg.MXFP4Weights(torch.zeros((2, 4, 33), dtype=torch.uint8, device=cuda), 64, 4)
    assert torch.isfinite(pkg.mxfp4_mul_mat_id(**good)).all()


@pytest.mark.parametrize("n", [2, 50, 300])
def test_captured_and_replayed(pkg, cuda, n):
    rng = np.random.default_rng(n)
    W = _experts(rng, 8, 200, 256)
    w = _weights(pkg, cuda, W, 256)
    x = torch.from_numpy(rng.normal(size=(n, 256)).astype(np.float32)).to(cuda)
    ids = torch.from_numpy(_ids(rng, n, 2, 8)).to(cuda)
    ws = torch.empty(pkg.mxfp4_workspace_size(w, n, 2), dtype=torch.uint8, device=cuda)
    pkg.mxfp4_mul_mat_id(w, x, ids, gate=w, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h = pkg.mxfp4_mul_mat_id(w, x, ids, gate=w, workspace=ws)
        y = pkg.mxfp4_mul_mat_id(w, x, ids, workspace=ws)          # behind the first, so they may share it
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        ids.copy_(torch.from_numpy(_ids(rng, n, 2, 8)).to(cuda))
        h.zero_()
        g.replay()
        assert torch.equal(h, pkg.mxfp4_mul_mat_id(w, x, ids, gate=w)) and torch.equal(y, pkg.mxfp4_mul_mat_id(w, x, ids))


def test_streams_side_by_side(pkg, cuda):
    """Calls on several streams at once, each with its own workspace, against the same calls alone."""
    rng = np.random.default_rng(3)
    w = _weights(pkg, cuda, _experts(rng, 16, 384, 512), 512)
    jobs = []
    for n in (1, 7, 30, 200, 64, 3):
        x = torch.from_numpy(rng.normal(size=(n, 512)).astype(np.float32)).to(cuda)
        jobs.append((x, torch.from_numpy(_ids(rng, n, 4, 16)).to(cuda)))
    alone = [pkg.mxfp4_mul_mat_id(w, x, ids, gate=w) for x, ids in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(20):
        got = [pkg.mxfp4_mul_mat_id(w, x, ids, gate=w, stream=s) for (x, ids), s in zip(jobs, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))
    assert pkg.moe_cache.device_error() == 0


@pytest.mark.parametrize("n", [2, 50, 300])
def test_waits_give_up(pkg, cuda, n):
    """A wait limit of 1 ns: the kernel gives up, reports it and leaves the context usable."""
    mc = pkg.moe_cache
    rng = np.random.default_rng(n)
    w = _weights(pkg, cuda, _experts(rng, 8, 256, 2048), 2048)
    x = torch.from_numpy(rng.normal(size=(n, 2048)).astype(np.float32)).to(cuda)
    ids = torch.from_numpy(_ids(rng, n, 2, 8)).to(cuda)
    good = pkg.mxfp4_mul_mat_id(w, x, ids, gate=w)
    assert mc.device_error() == 0
    try:
        mc.set_wait_limits(kernel_wait_ns=1)
        pkg.mxfp4_mul_mat_id(w, x, ids, gate=w)
        code = mc.device_error()
    finally:
        mc.set_wait_limits()
    assert code == mc.DERR_TIMEOUT_FULL
    assert torch.equal(pkg.mxfp4_mul_mat_id(w, x, ids, gate=w), good)
    assert mc.device_error() == 0


@pytest.mark.parametrize("n,k,E,K,rows,per_pick", [
    (3, 20, 40, 64, 33, False),        # more picks than a row's lanes look up at once, direct
    (40, 12, 700, 96, 70, False),      # and grouped, with one set of counters
    (30, 4, 4096, 32, 17, False),      # the most experts
    (16, 3, 4096, 64, 20, True),       # and direct
    (4500, 8, 16, 32, 20, False),      # entries past those whose ids stay in registers
    (33000, 1, 3, 32, 16, True),
    (2100, 16, 24, 96, 40, False),     # both
])
def test_product_of_many(pkg, cuda, n, k, E, K, rows, per_pick):
    rng = np.random.default_rng(n + E)
    W = _experts(rng, E, rows, K)
    x = rng.normal(size=(n, k, K) if per_pick else (n, K))
    ids = _ids(rng, n, k, E)
    ids[rng.random(ids.shape) < 0.05] = -1
    dst = torch.full((n, k, rows), 7.0, device=cuda)
    y, xv = _run(pkg, cuda, W, x, ids, K, 2, torch.float32, None, dst)
    assert pkg.moe_cache.device_error() == 0 and (y[ids < 0] == 7.0).all()
    ref, mag = R.product(W, xv, np.maximum(ids, 0), 2, None)
    assert (np.abs(y - ref) <= R.product_tol(mag, K, 2))[ids >= 0].all()


def test_offsets_past_32_bits(pkg, cuda):
    """Rows of x and of dst more than 2^31 elements from their tensors' first."""
    rng = np.random.default_rng(1)
    E, K, rows = 2, 64, 40
    W = _experts(rng, E, rows, K)
    w = _weights(pkg, cuda, W, K)
    n, wide = 70000, 32768
    big = torch.empty((n, wide), dtype=torch.bfloat16, device=cuda)          # 4.6 GB, 2.3e9 elements
    x = big[:, 8:8 + K]
    x.copy_(torch.randn((n, K), device=cuda))
    ids = torch.randint(0, E, (n, 1), dtype=torch.int32, device=cuda)
    tail = x[-64:].contiguous()
    assert torch.equal(pkg.mxfp4_mul_mat_id(w, x, ids)[-64:], pkg.mxfp4_mul_mat_id(w, tail, ids[-64:].contiguous()))
    assert torch.equal(pkg.quantize_mxfp4(x)[-64:], pkg.quantize_mxfp4(tail))
    assert torch.equal(pkg.route_experts(x, 4)[0][-64:], pkg.route_experts(tail, 4)[0])
    pkg.dequantize_mxfp4(pkg.quantize_mxfp4(tail), K, dtype=torch.bfloat16, out=x[-64:])
    assert torch.equal(x[-64:], pkg.dequantize_mxfp4(pkg.quantize_mxfp4(tail), K, dtype=torch.bfloat16))
    del big, x
    n, rows = 4200, 65536                                                    # dst: 8.8 GB, 2.2e9 elements
    W = _experts(rng, E, rows, 32)
    w = _weights(pkg, cuda, W, 32)
    x = torch.randn((n, 32), device=cuda)
    ids = torch.randint(0, E, (n, 8), dtype=torch.int32, device=cuda)
    y = pkg.mxfp4_mul_mat_id(w, x, ids)
    assert torch.equal(y[-8:], pkg.mxfp4_mul_mat_id(w, x[-8:].contiguous(), ids[-8:].contiguous()))


@pytest.mark.parametrize("n", [3, 120])
def test_two_graphs_at_once(pkg, cuda, n):
    """Two captured calls with workspaces of their own (a few tokens: none), replayed on two streams at once."""
    rng = np.random.default_rng(n)
    w = _weights(pkg, cuda, _experts(rng, 16, 384, 512), 512)
    xs = [torch.randn((n, 512), device=cuda) for _ in range(2)]
    ids = [torch.from_numpy(_ids(rng, n, 4, 16)).to(cuda) for _ in range(2)]
    alone = [pkg.mxfp4_mul_mat_id(w, x, i, gate=w) for x, i in zip(xs, ids)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, i in zip(xs, ids):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pkg.mxfp4_mul_mat_id(w, x, i, gate=w))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, alone))
    assert pkg.moe_cache.device_error() == 0
