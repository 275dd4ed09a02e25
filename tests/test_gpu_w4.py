"""Products with 4-bit matrices of group scales against the plain 64-bit
implementation (sorted_ref)."""
import numpy as np
import pytest
import torch

import sorted_ref as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Case:
    def __init__(self, pkg, cuda, rng, E, rows, K, group, zeros, scale="f16", flat=False):
        n = -(-K // group)
        self.K, self.group = K, group
        shape = (rows,) if flat else (E, rows)
        self.codes = rng.integers(0, 256, size=(*shape, (K + 1) // 2), dtype=np.uint8)
        s = torch.from_numpy((0.01 * (0.2 + rng.random((*shape, n))) * rng.choice([-1, 1], (*shape, n))).astype(np.float32)).to(DT[scale])
        self.zeros = rng.integers(0, 16, size=(*shape, n), dtype=np.uint8) if zeros else None
        self.scales = s.double().numpy()
        t = lambda a: None if a is None else torch.from_numpy(a).to(cuda)   # noqa: E731
        self.w = pkg.W4Weights(t(self.codes), s.to(cuda), K, group, zeros=t(self.zeros))
        self.values, self.parts = (v.reshape(E, rows, K) for v in R.w4_values(self.codes, self.scales, self.zeros, K, group))


def make_x(rng, shape, dtype, cuda):
    x = torch.from_numpy(rng.normal(size=shape).astype(np.float32)).to(cuda).to(DT[dtype])
    return x, x.double().cpu().numpy()


def product(c, x, ids):
    """([n, k, rows], the bound of its partial sums); x [n, K] or [n, k, K]"""
    n, k = ids.shape
    values, parts = c if isinstance(c, tuple) else (c.values, c.parts)
    x = np.broadcast_to(x[:, None], (n, k, x.shape[-1])) if x.ndim == 2 else x
    y, mag = (np.zeros((n, k, values.shape[1])) for _ in range(2))
    for t in range(n):
        for p in range(k):
            if 0 <= ids[t, p] < values.shape[0]:
                e = ids[t, p]
                y[t, p], mag[t, p] = values[e] @ x[t, p], parts[e] @ np.abs(x[t, p])
    return y, mag


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,rows,K,group,zeros", [
    (1, 1, 1, 32, False), (1, 16, 64, 64, True), (1, 17, 33, 32, True), (2, 30, 31, 32, False), (3, 100, 96, 32, True),
    (1, 768, 2048, 128, False), (5, 1000, 1446, 128, True), (7, 40, 700, 1024, True), (4, 64, 999, 256, False),
    (8, 33, 4096, 32, True), (9, 129, 512, 64, False), (16, 48, 1024, 128, True), (17, 50, 2000, 64, True),
    (24, 256, 4096, 32, True), (33, 20, 320, 128, False), (70, 130, 640, 64, True), (2, 5000, 128, 32, True),
    (11, 64, 20000, 128, True), (32, 64, 9000, 32, False),                       # K in several passes
])
def test_one_matrix(pkg, cuda, n, rows, K, group, zeros, dtype):
    rng = np.random.default_rng(rows + K)
    c = Case(pkg, cuda, rng, 1, rows, K, group, zeros, scale=("f16", "bf16")[n % 2], flat=n % 2 == 0)
    x, x64 = make_x(rng, (n, K), dtype, cuda)
    got = pkg.w4_mul_mat(c.w, x).double().cpu().numpy()
    ref, mag = product(c, x64, np.zeros((n, 1), np.int32))
    assert got.shape == (n, rows)
    err = np.abs(got - ref[:, 0])
    assert (err <= R.w4_tol(mag[:, 0], K)).all(), (err / R.w4_tol(mag[:, 0], K)).max()
    assert pkg.moe_cache.device_error() == 0


EXPERTS = [
    # n, E, k, rows, K, group, zeros, per_pick
    (1, 8, 4, 48, 256, 128, False, False), (1, 4, 4, 20, 64, 32, True, True), (3, 5, 2, 100, 1446, 64, True, False),
    (8, 64, 8, 64, 768, 32, False, True), (16, 3, 4, 33, 512, 128, True, False),        # 64 picks: grouped in the kernel
    (13, 3, 5, 33, 512, 128, True, True), (64, 16, 8, 96, 448, 64, False, False), (100, 2, 3, 40, 320, 32, True, True),
    (40, 300, 6, 16, 96, 32, False, False), (5, 1, 1, 31, 62, 32, True, False), (90, 1, 1, 31, 62, 64, True, False),
    (12, 4, 5, 24, 6000, 128, True, False),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,E,k,rows,K,group,zeros,per_pick", EXPERTS)
def test_experts(pkg, cuda, n, E, k, rows, K, group, zeros, per_pick, dtype):
    """Picks dropped and repeated; their rows of dst stay as they were; biases."""
    rng = np.random.default_rng(n + E + K)
    c = Case(pkg, cuda, rng, E, rows, K, group, zeros, scale=("f16", "bf16")[E % 2])
    ids = rng.integers(0, E, size=(n, k)).astype(np.int32)
    ids[rng.random((n, k)) < 0.15] = -1
    x, x64 = make_x(rng, (n, k, K) if per_pick else (n, K), dtype, cuda)
    bias = rng.normal(size=(E, rows)).astype(np.float32)
    dst = torch.full((n, k, rows), 7.25, device=cuda)
    tids = torch.from_numpy(ids).to(cuda)
    got = pkg.w4_mul_mat_id(c.w, x, tids, bias=torch.from_numpy(bias).to(cuda), dst=dst)
    assert got is dst
    got = got.double().cpu().numpy()
    ref, mag = product(c, x64, ids)
    held = ids >= 0
    assert (got[~held] == 7.25).all()
    b = bias.astype(np.float64)[np.maximum(ids, 0)]
    assert (np.abs(got - ref - b)[held] <= R.w4_tol(mag + np.abs(b), K)[held]).all()
    again = pkg.w4_mul_mat_id(c.w, x, tids, bias=torch.from_numpy(bias).to(cuda))
    assert torch.equal(again[tids >= 0], dst[tids >= 0])
    assert pkg.moe_cache.device_error() == 0


@pytest.mark.parametrize("op", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("n,E,k,rows,K,group,zeros,dtype,biases", [
    (1, 8, 4, 100, 2048, 128, False, "f32", False), (9, 3, 4, 40, 320, 32, True, "f16", True), (30, 5, 3, 33, 700, 64, True, "bf16", True),
    (20, 2, 2, 64, 9000, 128, False, "bf16", True), (2, 1, 1, 64, 5000, 32, True, "f32", False),
])
def test_gate(pkg, cuda, n, E, k, rows, K, group, zeros, dtype, biases, op):
    rng = np.random.default_rng(K + op)
    up, gate = (Case(pkg, cuda, rng, E, rows, K, group, zeros) for _ in range(2))
    ids = rng.integers(0, E, size=(n, k)).astype(np.int32)
    x, x64 = make_x(rng, (n, K), dtype, cuda)
    b = [rng.normal(size=(E, rows)).astype(np.float32) if biases else np.zeros((E, rows), np.float32) for _ in range(2)]
    kw = dict(bias=torch.from_numpy(b[0]).to(cuda), gate_bias=torch.from_numpy(b[1]).to(cuda)) if biases else {}
    if E == 1:
        got = pkg.w4_mul_mat(up.w, x, gate=gate.w, glu_op=op, glu_limit=1.25, **kw)[:, None]
    else:
        got = pkg.w4_mul_mat_id(up.w, x, torch.from_numpy(ids).to(cuda), gate=gate.w, glu_op=op, glu_limit=1.25, **kw)
    (u, mu), (g, mg) = (product(c, x64, ids) for c in (up, gate))
    u, g = u + b[0].astype(np.float64)[ids], g + b[1].astype(np.float64)[ids]
    eu, eg = R.w4_tol(mu + np.abs(b[0])[ids], K), R.w4_tol(mg + np.abs(b[1])[ids], K)
    err = np.abs(got.double().cpu().numpy() - R.glu(op, g, u, 1.25))
    assert (err <= R.glu_tol(op, g, u, eg, eu, 1.25)).all()


def test_exact_values(pkg, cuda):
    """Every code against every zero, scales that are powers of two, x a unit vector: the values come back exactly."""
    K, rows = 64, 128
    codes = np.tile((np.arange(32, dtype=np.uint8) * 2 % 16) | ((np.arange(32, dtype=np.uint8) * 2 + 1) % 16 << 4), (rows, 1))
    zeros = np.stack([np.arange(rows), 127 - np.arange(rows)], 1).astype(np.uint8)
    scales = np.exp2((np.arange(rows * 2) % 7 - 3).reshape(rows, 2)).astype(np.float16)
    ref = R.w4_values(codes, scales.astype(np.float64), zeros, K, 32)[0]
    t = lambda a: torch.from_numpy(a).to(cuda)   # noqa: E731
    w = pkg.W4Weights(t(codes), t(scales), K, 32, zeros=t(zeros))
    assert pkg.moe_cache.device_error() == 0
    for dt in DT.values():
        np.testing.assert_array_equal(pkg.w4_mul_mat(w, torch.eye(K, device=cuda, dtype=dt)).cpu().numpy().T, ref)


def test_x_of_32_bits(pkg, cuda):
    """x of full 24-bit mantissas over the exponents that products leave finite, one value in 256: two planes hold it to
    2^-22, and (9 - 8) x costs one rounding of 9 x and one of the difference more."""
    K = 300
    codes = torch.full((16, 150), 0x99, dtype=torch.uint8, device=cuda)          # q - 8 = 1
    w = pkg.W4Weights(codes, torch.full((16, 1), 0.5, dtype=torch.float16, device=cuda), K, 512)
    rng = np.random.default_rng(1)
    x = torch.zeros((200, K), device=cuda)
    vals = (rng.uniform(1, 2, 200) * np.exp2(rng.integers(-100, 120, 200)) * rng.choice([-1, 1], 200)).astype(np.float32)
    for i, v in enumerate(vals):
        x[i, i] = float(v)
    y = pkg.w4_mul_mat(w, x).double().cpu().numpy()
    want = np.repeat(vals[:, None].astype(np.float64) * 0.5, 16, 1)
    assert (np.abs(y - want) <= (2.0 ** -22 + 18 * 2.0 ** -24) * np.abs(want)).all()


def test_bf16_over_its_range(pkg, cuda):
    """bf16 values 2^24 apart in one block are exact; below 2^-39 of the block's largest nothing is left of them."""
    K = 256
    codes = torch.full((16, 128), 0x88, dtype=torch.uint8, device=cuda)          # 0,
    codes[:, 1:] = 0x98                                                          # and 0, 1 from the third value on
    w = pkg.W4Weights(codes, torch.ones((16, 1), dtype=torch.float16, device=cuda), K, 256)
    for p in (-90, 0, 100):
        for d in (1, 10, 24, 28):
            x = torch.zeros((1, K), device=cuda, dtype=torch.bfloat16)
            x[0, 0], x[0, 3] = 1.5 * 2.0 ** p, -1.25 * 2.0 ** (p - d)
            y = pkg.w4_mul_mat(w, x).double().cpu()
            # sums of q x: 8 * 1.5 and 9 * 1.25 2^-d against 8 times their sum, in 32 bits
            assert ((y + 1.25 * 2.0 ** (p - d)).abs() <= 3 * 24.0 * 2.0 ** (p - 24)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_nan_and_inf_stay_in_their_row(pkg, cuda, dtype):
    rng = np.random.default_rng(2)
    for n, K in ((12, 300), (2, 70), (12, 3000)):
        c = Case(pkg, cuda, rng, 1, 70, K, 64, True)
        x, _ = make_x(rng, (n, K), dtype, cuda)
        good = pkg.w4_mul_mat(c.w, x)
        hit = {0: float("nan")} if n < 3 else {3: float("nan"), 5: float("inf"), 8: float("-inf")}
        for i, (row, v) in enumerate(hit.items()):
            x[row, (17, K - 1, 0)[i]] = v
        y = pkg.w4_mul_mat(c.w, x)
        assert all(torch.isnan(y[row]).all() for row in hit)
        rest = [i for i in range(n) if i not in hit]
        assert torch.equal(y[rest], good[rest])


def test_bad_ids_and_zeros(pkg, cuda):
    mc = pkg.moe_cache
    rng = np.random.default_rng(3)
    c = Case(pkg, cuda, rng, 4, 40, 128, 64, True)
    for n in (3, 60):                                                            # both forms
        x, x64 = make_x(rng, (n, 128), "f32", cuda)
        ids = rng.integers(0, 4, size=(n, 2)).astype(np.int32)
        for bad in (4, -2, 2 ** 31 - 1, -2 ** 31):
            ids[1, 1] = bad
            dst = torch.full((n, 2, 40), 3.5, device=cuda)
            pkg.w4_mul_mat_id(c.w, x, torch.from_numpy(ids).to(cuda), dst=dst)
            assert mc.device_error() == mc.DERR_BAD_ID and mc.device_error() == 0
            assert (dst[1, 1] == 3.5).all()
            ref, mag = product(c, x64, ids)
            ok = ids < 4
            ok[1, 1] = False
            assert (np.abs(dst.double().cpu().numpy() - ref)[ok] <= R.w4_tol(mag, 128)[ok]).all()
        none = torch.full((n, 2), -1, dtype=torch.int32, device=cuda)
        dst = torch.full((n, 2, 40), 3.5, device=cuda)
        assert (pkg.w4_mul_mat_id(c.w, x, none, dst=dst) == 3.5).all()
    zeros = torch.full((16, 1), 128, dtype=torch.uint8, device=cuda)
    pkg.W4Weights(torch.zeros((16, 16), dtype=torch.uint8, device=cuda), torch.ones((16, 1), dtype=torch.float16, device=cuda),
                  32, 32, zeros=zeros)
    assert mc.device_error() == mc.DERR_BAD_ZERO


def test_rows_of_wider_buffers(pkg, cuda):
    rng = np.random.default_rng(4)
    c = Case(pkg, cuda, rng, 3, 50, 320, 64, False)
    for dtype in DT:
        big, _ = make_x(rng, (20, 320 + 24), dtype, cuda)
        ids = torch.from_numpy(rng.integers(0, 3, size=(20, 9)).astype(np.int32)).to(cuda)
        for at in (0, 1, 8, 24):
            for sl in (ids[:, :4], ids[:, 3:5], ids[:3, 2:7]):
                x = big[: sl.shape[0], at:at + 320]
                assert torch.equal(pkg.w4_mul_mat_id(c.w, x, sl), pkg.w4_mul_mat_id(c.w, x.contiguous(), sl.contiguous()))


def test_streams_and_graphs(pkg, cuda):
    rng = np.random.default_rng(5)
    c = Case(pkg, cuda, rng, 6, 80, 512, 128, True)
    for n, k in ((4, 2), (50, 3)):
        x, _ = make_x(rng, (n, 512), "bf16", cuda)
        ids = torch.from_numpy(rng.integers(0, 6, size=(n, k)).astype(np.int32)).to(cuda)
        want = pkg.w4_mul_mat_id(c.w, x, ids)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        for stream in (s, s.cuda_stream):
            y = pkg.w4_mul_mat_id(c.w, x, ids, stream=stream)
            s.synchronize()
            assert torch.equal(y, want)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = pkg.w4_mul_mat_id(c.w, x, ids)
            graphs.append((g, y))
        x.neg_()
        torch.cuda.synchronize()
        for g, y in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        torch.cuda.synchronize()
        for g, y in graphs:
            assert torch.equal(y, -want)
    assert pkg.moe_cache.device_error() == 0


def test_a_token_alone_and_in_a_batch(pkg, cuda):
    """A token's result depends on its own row: the same bits wherever the call's sums of a row have the same order
    (they do: K is shared by the same warps whatever the batch; passes of K add their sums apart)."""
    rng = np.random.default_rng(6)
    c = Case(pkg, cuda, rng, 1, 64, 512, 64, True)
    x, _ = make_x(rng, (40, 512), "bf16", cuda)
    all_of = pkg.w4_mul_mat(c.w, x)
    for i in (0, 7, 39):
        assert torch.equal(pkg.w4_mul_mat(c.w, x[i:i + 1])[0], all_of[i])


def test_no_tokens(pkg, cuda):
    rng = np.random.default_rng(7)
    c = Case(pkg, cuda, rng, 2, 16, 64, 64, False)
    x = torch.empty((0, 64), device=cuda)
    assert pkg.w4_mul_mat_id(c.w, x, torch.empty((0, 3), dtype=torch.int32, device=cuda)).shape == (0, 3, 16)


@pytest.mark.parametrize("n", [1, 70])
def test_routed_experts_sorted_and_combined(pkg, cuda, n):
    """A layer out of the pieces: route, then either the experts' products by pick, or rows sorted by expert, their
    products (one pick a row), and the weighted sum back."""
    rng = np.random.default_rng(8)
    H, F, E, k = 256, 96, 16, 4
    up, gate, down = (Case(pkg, cuda, rng, E, r, K, 64, True) for r, K in ((F, H), (F, H), (H, F)))
    x, x64 = make_x(rng, (n, H), "f32", cuda)
    shared, s64 = make_x(rng, (n, H), "f32", cuda)
    logits = torch.from_numpy(rng.normal(size=(n, E)).astype(np.float32)).to(cuda)
    ids, w = pkg.Router(k, norm_w=True)(logits)
    rows, order = pkg.dispatch_sorted(x, ids, E)
    one = order.experts.view(-1, 1)
    h = pkg.w4_mul_mat_id(up.w, rows, one, gate=gate.w)[:, 0]
    y = pkg.w4_mul_mat_id(down.w, h, one)[:, 0]
    out = pkg.combine_sorted(y, order, w, shared=shared)
    hp = pkg.w4_mul_mat_id(up.w, x, ids, gate=gate.w)
    yp = pkg.w4_mul_mat_id(down.w, hp, ids)
    assert torch.equal(h[order.positions.long()], hp) and torch.equal(y[order.positions.long()], yp)
    i, w64 = ids.cpu().numpy(), w.double().cpu().numpy()
    (u, mu), (g, mg) = (product(c, x64, i) for c in (up, gate))
    ref_h = R.glu(0, g, u)
    eh = R.glu_tol(0, g, u, R.w4_tol(mg, H), R.w4_tol(mu, H))
    ref_y, mag = product(down, ref_h, i)
    ey = R.w4_tol(mag, F) + product((np.abs(down.values), down.parts), eh, i)[0]
    ref = (ref_y * w64[..., None]).sum(1) + s64
    parts = np.abs(ref_y * w64[..., None]).sum(1) + np.abs(s64)
    tol = (ey * w64[..., None]).sum(1) * 1.01 + R.combine_tol(ref, parts, k, "f32")
    assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all()
    assert pkg.moe_cache.device_error() == 0


def test_calls_behind_one_another_and_at_once(pkg, cuda):
    """Calls that overlap: each one's x is the result before it, and its ids those of an order; on two streams at a time."""
    rng = np.random.default_rng(9)
    E, F, H, k = 12, 160, 320, 3
    up, down = Case(pkg, cuda, rng, E, F, H, 64, True), Case(pkg, cuda, rng, E, H, F, 32, False)
    one = Case(pkg, cuda, rng, 1, H, H, 128, False)
    sets = []
    for n in (1, 30, 400):
        x, _ = make_x(rng, (n, H), "f32", cuda)
        sets.append((x, torch.from_numpy(rng.integers(0, E, size=(n, k)).astype(np.int32)).to(cuda)))

    def chain(x, ids, wait=lambda: None):
        for _ in range(3):
            rows, order = pkg.dispatch_sorted(x, ids, E)
            wait()
            ex = order.experts.view(-1, 1)
            h = pkg.w4_mul_mat_id(up.w, rows, ex)[:, 0]
            wait()
            y = pkg.w4_mul_mat_id(down.w, h, ex)[:, 0]
            wait()
            x = pkg.combine_sorted(y, order, torch.full(ids.shape, 1.0 / k, device=cuda))
            wait()
            x = pkg.w4_mul_mat(one.w, x)
            wait()
            x = x / x.abs().amax()
        return x
    want = [chain(*s, wait=torch.cuda.synchronize) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(chain(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [chain(*s) for s in sets]
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    assert pkg.moe_cache.device_error() == 0


def test_given_workspaces(pkg, cuda):
    rng = np.random.default_rng(10)
    c, one = Case(pkg, cuda, rng, 5, 70, 300, 64, True), Case(pkg, cuda, rng, 1, 70, 300, 64, True)
    for n, k, per_pick in ((40, 2, False), (600, 2, True)):
        x, _ = make_x(rng, (n, k, 300) if per_pick else (n, 300), "bf16", cuda)
        ids = torch.from_numpy(rng.integers(0, 5, size=(n, k)).astype(np.int32)).to(cuda)
        need = pkg.w4_workspace_size(c.w, n, k, x.dtype, per_pick)
        assert need > 0
        ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=cuda)
        assert torch.equal(pkg.w4_mul_mat_id(c.w, x, ids, workspace=ws[:need]), pkg.w4_mul_mat_id(c.w, x, ids))
        assert (ws[need:] == 255).all()
        with pytest.raises(pkg.MoeError, match="too small"):
            pkg.w4_mul_mat_id(c.w, x, ids, workspace=ws[: need - 16])
        with pytest.raises(pkg.MoeError, match="aligned"):
            pkg.w4_mul_mat_id(c.w, x, ids, workspace=ws[1: need + 1])
    x, _ = make_x(rng, (40, 300), "f32", cuda)
    ws = torch.empty(pkg.w4_workspace_size(one.w, 40, 0, x.dtype), dtype=torch.uint8, device=cuda)
    assert torch.equal(pkg.w4_mul_mat(one.w, x, workspace=ws), pkg.w4_mul_mat(one.w, x))


def test_many_experts_and_picks(pkg, cuda):
    """1024 experts; 1024 picks, the last that every CTA groups by itself, and the first that a launch of its own does."""
    rng = np.random.default_rng(11)
    c = Case(pkg, cuda, rng, 1024, 16, 32, 32, False)
    for n, k in ((512, 2), (205, 5), (1024, 1), (1, 1)):
        ids = rng.integers(0, 1024, size=(n, k)).astype(np.int32)
        x, x64 = make_x(rng, (n, 32), "f16", cuda)
        got = pkg.w4_mul_mat_id(c.w, x, torch.from_numpy(ids).to(cuda)).double().cpu().numpy()
        ref, mag = product(c, x64, ids)
        assert (np.abs(got - ref) <= R.w4_tol(mag, 32)).all()


def test_offsets_past_32_bits(pkg, cuda):
    """Matrices of more than 2^32 bytes: the last experts' values."""
    E, rows, K = 600, 2048, 8192
    g = torch.Generator(device=cuda).manual_seed(1)
    codes = torch.empty((E, rows, K // 2), dtype=torch.uint8, device=cuda)
    codes.random_(0, 256, generator=g)
    scales = torch.full((E, rows, K // 256), 0.01, dtype=torch.bfloat16, device=cuda)
    w = pkg.W4Weights(codes, scales, K, 256)
    x = torch.randn((2, K), generator=g, device=cuda)
    ids = torch.tensor([[E - 1, 0], [E - 2, E // 2]], dtype=torch.int32, device=cuda)
    y = pkg.w4_mul_mat_id(w, x, ids)
    for t in range(2):
        for p in range(2):
            e = int(ids[t, p])
            q = torch.stack([codes[e] & 15, codes[e] >> 4], -1).view(rows, K).double()
            s = float(torch.tensor(0.01, dtype=torch.bfloat16))
            ref, mag = ((q - 8) * s) @ x[t].double(), ((q + 8) * s) @ x[t].double().abs()
            assert ((y[t, p].double() - ref).abs().cpu().numpy() <= R.w4_tol(mag.cpu().numpy(), K)).all()


def test_refusals(pkg, cuda):
    codes, scales = torch.zeros((3, 8, 32), dtype=torch.uint8, device=cuda), torch.ones((3, 8, 2), dtype=torch.float16, device=cuda)
    zeros = torch.zeros((3, 8, 2), dtype=torch.uint8, device=cuda)
    W = pkg.W4Weights
    w, one = W(codes, scales, 64, 32), W(codes[0], scales[0], 64, 32)
    x, ids = torch.zeros((4, 64), device=cuda), torch.zeros((4, 2), dtype=torch.int32, device=cuda)
    b = torch.zeros((3, 8), device=cuda)
    for f in (lambda: W(codes.int(), scales, 64, 32), lambda: W(codes, scales.float(), 64, 32), lambda: W(codes, scales, 66, 32),
              lambda: W(codes, scales, 64, 64), lambda: W(codes, scales, 64, 16), lambda: W(codes, scales[:2], 64, 32),
              lambda: W(codes, scales, 64, 32, zeros=zeros.float()), lambda: W(codes, scales, 64, 32, zeros=zeros[..., :1]),
              lambda: W(codes[..., ::2], scales, 32, 32), lambda: W(codes[0, 0], scales[0, 0], 64, 32),
              lambda: pkg.w4_mul_mat(w, x), lambda: pkg.w4_mul_mat(one, x[:, :32]), lambda: pkg.w4_mul_mat(one, x.double()),
              lambda: pkg.w4_mul_mat(one, x[0]), lambda: pkg.w4_mul_mat(one, x, gate=w), lambda: pkg.w4_mul_mat(one, x, gate_bias=b[:1]),
              lambda: pkg.w4_mul_mat(one, x, bias=b), lambda: pkg.w4_mul_mat(one, x, dst=torch.empty((4, 8), device=cuda, dtype=torch.float16)),
              lambda: pkg.w4_mul_mat(one, x, gate=W(codes[0], scales[0], 64, 32, zeros=zeros[0])), lambda: pkg.w4_mul_mat(one, x, gate=one, glu_op=9),
              lambda: pkg.w4_mul_mat_id(w, x, ids.long()), lambda: pkg.w4_mul_mat_id(w, x[:3], ids), lambda: pkg.w4_mul_mat_id(w, x, ids[0]),
              lambda: pkg.w4_mul_mat_id(w, x, ids, bias=b[:2]), lambda: pkg.w4_mul_mat_id(w, x, ids, bias=b.half()),
              lambda: pkg.w4_mul_mat_id(w, x.cpu(), ids), lambda: pkg.w4_mul_mat_id(w, x, ids, dst=torch.empty((4, 2, 9), device=cuda)),
              lambda: pkg.w4_mul_mat_id(w, x, ids, workspace=torch.empty(4, device=cuda))):
        with pytest.raises(pkg.MoeError):
            f()
    assert pkg.w4_mul_mat(one, x, bias=b[0]).shape == pkg.w4_mul_mat(one, x, bias=b[:1]).shape == (4, 8)
    assert pkg.moe_cache.device_error() == 0


def test_products_right_behind_the_packing(pkg, cuda):
    """Equal bits with and without a pause between the layout of the matrix and its first products, in a graph too."""
    rng = np.random.default_rng(21)
    rows, K, group = 4096, 4096, 128
    t = lambda a: torch.from_numpy(a).to(cuda)   # noqa: E731
    codes = [t(rng.integers(0, 256, size=(rows, K // 2), dtype=np.uint8)) for _ in range(3)]
    scales = t((0.01 * rng.random((rows, K // group))).astype(np.float16))
    xs = [make_x(rng, (n, K), "f16", cuda)[0] for n in (1, 24)]       # 24: x is staged by a launch between

    def products(q, pause=False):
        w = pkg.W4Weights(q, scales, K, group)
        if pause:
            torch.cuda.synchronize()
        return [pkg.w4_mul_mat(w, x) for x in (*xs, *xs[::-1])]
    want = [products(q, True) for q in codes]
    torch.cuda.synchronize()
    for _ in range(4):
        got = [products(q) for q in codes]         # the memory of one matrix is the next one's
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(want, got) for a, b in zip(p, q))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = [products(q) for q in codes]
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for p, q in zip(want, got) for a, b in zip(p, q))
    assert pkg.moe_cache.device_error() == 0
