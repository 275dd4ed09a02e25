"""Products with 4-bit matrices in every form that the plan has, against 64-bit products: each element, and the 2-norm."""
import numpy as np
import pytest
import torch

import sorted_ref as R
import w4_forms as F

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Matrices:
    def __init__(self, pkg, cuda, g, E, rows, K, group, zeros, flat):
        shape, n = (rows,) if flat else (E, rows), -(-K // group)
        self.codes = torch.randint(0, 256, (*shape, (K + 1) // 2), generator=g, device=cuda, dtype=torch.uint8)
        self.scales = (0.01 * (0.2 + torch.rand((*shape, n), generator=g, device=cuda))).to(DT["bf16" if zeros else "f16"])
        self.zeros = torch.randint(0, 16, (*shape, n), generator=g, device=cuda, dtype=torch.uint8) if zeros else None
        self.w = pkg.W4Weights(self.codes, self.scales, K, group, zeros=self.zeros)
        self.K, self.group, self.flat = K, group, flat

    def values(self, e):
        """(s (q - z), |s| (q + z)) of a matrix, f64 [rows, K]"""
        codes, scales, zeros = (m if m is None or self.flat else m[e] for m in (self.codes, self.scales, self.zeros))
        at = torch.arange(self.K, device=codes.device) // self.group
        q = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1)[:, : self.K].double()
        z = 8.0 if zeros is None else zeros.double()[:, at]
        return (q - z) * scales.double()[:, at], (q + z) * scales.double().abs()[:, at]

    def product(self, x, ids):
        """[n, k, rows] and the sums of magnitudes, f64; x [n, K]"""
        y, mag = (torch.zeros((*ids.shape, self.w.rows), dtype=torch.float64, device=x.device) for _ in range(2))
        for e in ids.unique().tolist():
            if e >= 0:
                t, p = torch.nonzero(ids == e, as_tuple=True)
                v, parts = self.values(e)
                y[t, p], mag[t, p] = x[t].double() @ v.t(), x[t].double().abs() @ parts.t()
        return y, mag


def tol(mag, K):
    """w4_tol's, for K shared by up to 16 warps and 4 CTAs in up to 5 passes (8 additions more than it counts)"""
    return torch.from_numpy(R.w4_tol(mag.cpu().numpy(), K)).to(mag.device) + 8 * 2.0 ** -24 * mag


def norm(t):
    return float(torch.linalg.vector_norm(t))


@pytest.mark.parametrize("case", F.CASES, ids=lambda c: "-".join(str(int(v) if isinstance(v, bool) else v) for v in (*c[0], *c[1:])))
def test_form(pkg, cuda, case):
    want, rows, K, group, zeros, dtype, n, E, k, gate = case
    assert F.form(pkg, case) == want
    g = torch.Generator(device=cuda).manual_seed(rows + K + n)
    up = Matrices(pkg, cuda, g, E, rows, K, group, zeros, k == 0)
    gt = Matrices(pkg, cuda, g, E, rows, K, group, zeros, k == 0) if gate else None
    x = torch.randn((n, K), generator=g, device=cuda).to(DT[dtype])
    ids = torch.randint(0, E, (n, max(1, k)), generator=g, device=cuda, dtype=torch.int32)
    held = torch.ones_like(ids, dtype=torch.bool)
    kw = dict(gate=gt.w, glu_op=pkg.moe_cache.GLU_PRODUCT) if gate else {}
    if k:
        held = torch.rand(ids.shape, generator=g, device=cuda) > 0.1
        held[0, 0] = True
        ids[~held] = -1
        dst = torch.full((n, k, rows), 7.25, device=cuda)
        got = pkg.w4_mul_mat_id(up.w, x, ids, dst=dst, **kw)
        again = pkg.w4_mul_mat_id(up.w, x, ids, **kw)
        assert (got[~held] == 7.25).all()
    else:
        got, again = (pkg.w4_mul_mat(up.w, x, **kw)[:, None] for _ in range(2))
    assert torch.equal(got[held], again[held])
    ref, mag = up.product(x, ids)
    bound, factor = tol(mag, K), 1.0
    if gate:      # of a product of both: |du g| + |u dg| + |du dg|, and its own rounding
        rg, mg = gt.product(x, ids)
        bg = tol(mg, K)
        bound = bound * rg.abs() + bg * ref.abs() + bound * bg + 2.0 ** -24 * (ref * rg).abs()
        ref, factor = ref * rg, 2.0
    err = got.double() - ref
    assert (err.abs() <= bound)[held].all()
    assert norm(err[held]) <= factor * R.W4_NORM * norm(ref[held])
    assert pkg.moe_cache.device_error() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group,zeros", [(128, False), (32, True)])
def test_tokens_alone_and_in_batches(pkg, cuda, dtype, group, zeros):
    """The order of a row's sums goes with the number of tokens: results differ between batches, by roundings only."""
    g = torch.Generator(device=cuda).manual_seed(group)
    m = Matrices(pkg, cuda, g, 1, 4096, 4096, group, zeros, True)
    x = torch.randn((64, 4096), generator=g, device=cuda).to(DT[dtype])
    ref, mag = m.product(x, torch.zeros((64, 1), dtype=torch.int32, device=cuda))
    ref, bound, plans = ref[:, 0], tol(mag[:, 0], 4096), set()
    for n in (1, 2, 8, 24, 40, 64):
        plans.add(tuple(F.plan(pkg, 4096, 4096, group, zeros, dtype, n, 1, 0, False)))
        err = pkg.w4_mul_mat(m.w, x[:n]).double() - ref[:n]
        assert (err.abs() <= bound[:n]).all() and norm(err) <= R.W4_NORM * norm(ref[:n])
    assert len({p[2] for p in plans}) > 1          # K shared by more and by fewer warps


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,rows,K,group,zeros", [(1, 768, 2048, 128, False), (5, 1000, 1446, 128, True), (24, 4096, 4096, 32, True),
                                                  (1, 8192, 4096, 64, True), (9, 2048, 768, 32, False), (300, 1024, 2048, 128, True)])
def test_norms(pkg, cuda, n, rows, K, group, zeros, dtype):
    g = torch.Generator(device=cuda).manual_seed(n + rows)
    m = Matrices(pkg, cuda, g, 1, rows, K, group, zeros, True)
    x = torch.randn((n, K), generator=g, device=cuda).to(DT[dtype])
    ref = m.product(x, torch.zeros((n, 1), dtype=torch.int32, device=cuda))[0][:, 0]
    assert norm(pkg.w4_mul_mat(m.w, x).double() - ref) <= R.W4_NORM * norm(ref)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_small_values_next_to_large_ones(pkg, cuda, dtype):
    """Values 2^d below the largest of their 256, which meets code 0 and zero 0: x is held to 2^-39 of the largest (f16's least
    step 2^-24, half of it, under 2^14 to 2^15), and nothing else is rounded but the 32-bit result."""
    K, rows = 256, 16
    codes = torch.zeros((rows, K // 2), dtype=torch.uint8, device=cuda)
    codes[:, 1:] = 0x11
    w = pkg.W4Weights(codes, torch.ones((rows, 1), dtype=torch.float16, device=cuda), K, K,
                      zeros=torch.zeros((rows, 1), dtype=torch.uint8, device=cuda))
    for p in (-60, 0, 100):
        for d in (1, 8, 15, 20, 24, 28, 32, 36, 38):
            x = torch.zeros((1, K), device=cuda, dtype=DT[dtype])
            x[0, 0], x[0, 77] = 1.5 * 2.0 ** p, -1.25 * 2.0 ** (p - d)
            y = pkg.w4_mul_mat(w, x).double()
            want = -1.25 * 2.0 ** (p - d)
            assert ((y - want).abs() <= 2.0 ** -39 * 1.5 * 2.0 ** p + 2.0 ** -24 * abs(want)).all(), (p, d, float(y[0, 0]), want)
            assert (y[0, 0] == y[0]).all()


def test_large_values_on_their_zeros(pkg, cuda):
    """What the bound is relative to: a large x whose code is its zero adds nothing, but for roundings of code * x."""
    K = 2048
    g = torch.Generator(device=cuda).manual_seed(3)
    m = Matrices(pkg, cuda, g, 1, 64, K, 64, True, True)
    m.codes[:, 100] = m.zeros[:, 200 // 64] * 0x11
    m.w = pkg.W4Weights(m.codes, m.scales, K, 64, zeros=m.zeros)
    for size in (1.0, 2.0 ** 8, 2.0 ** 16, 2.0 ** 24):
        x = torch.randn((3, K), generator=g, device=cuda)
        x[:, 200:202] *= size
        ref, mag = m.product(x, torch.zeros((3, 1), dtype=torch.int32, device=cuda))
        assert ((pkg.w4_mul_mat(m.w, x).double() - ref[:, 0]).abs() <= tol(mag[:, 0], K)).all()
