"""The plans of products with 4-bit matrices, and the bounds that their tests use, on the CPU."""
import ctypes
from importlib import import_module

import numpy as np

import sorted_ref as R
import w4_forms as F

P = 0x1000


def test_the_cases_take_every_form(pkg):
    took = set()
    for case in F.CASES:
        assert F.form(pkg, case, F.B200) == case[0], case
        took.add((*case[0], case[8] > 0, case[9]))
    # (several passes of 8 columns for one matrix: only with clusters, at the sizes that were looked at)
    want = {(nt, split, passes, ids, gate) for nt in (1, 2) for split in (1, 2, 4) for passes in (False, True) for ids in (False, True)
            for gate in (False, True)} - {(1, 1, True, False, False), (1, 1, True, False, True), (1, 2, True, False, True)}
    assert took == want


def test_clusters_run_at_once(pkg):
    """148 SMs hold 33 clusters of 4, as clusters do not span GPCs: 34 to 37 of them would run in two rounds."""
    counted = 0
    for dtype, n, K, rows, group, zeros in (("f16", 16, 6968, 3718, 128, True), ("f32", 21, 7240, 732, 128, True), ("bf16", 49, 7206, 1368, 128, True),
                                            ("f16", 7, 7676, 3990, 64, True), ("f32", 24, 5086, 1952, 256, False), ("f16", 7, 7958, 5269, 128, False),
                                            ("f32", 14, 7796, 1718, 256, False), ("bf16", 8, 14336, 4096, 128, True), ("bf16", 1, 8192, 1024, 128, False)):
        for slots in (F.B200, (148, 74, 37), (148, 74, 0), (148, 0, 0)):
            nt, split, _, wm, _, _ = F.plan(pkg, rows, K, group, zeros, dtype, n, 1, 0, False, slots)
            chunks = -(-n // (8 * nt // (2 if dtype == "f32" else 1)))
            blocks = chunks * -(-(-(-rows // 16)) // wm)
            assert split == 1 or slots[split // 2] > 0
            if slots == F.B200 and split == 4:
                assert blocks <= 33
            counted += slots[2] == 37 and split == 4 and 33 < blocks <= 37
    assert counted >= 5       # what a count of 37 takes


def test_plan_arguments(pkg):
    lm = import_module("a6000-custom-kernels_b200._lib")
    out = (ctypes.c_int32 * 6)()

    def call(n=1, k=2, t=0, slots=F.B200, o=out, **kw):
        w = dict(E=2, rows=16, K=64, group=32, scale=1) | kw
        return pkg.lib().moe_b200_w4_plan(ctypes.byref(lm.MoeW4(None, w["E"], w["rows"], w["K"], w["group"], w["scale"], 0)), 0, n, k, t,
                                          (ctypes.c_int32 * 3)(*slots), o)
    assert call() == 0 and list(out)[:2] == [1, 1] and out[4] == 1
    assert call(n=0) == call(k=-1) == call(slots=(0, 0, 0)) == call(o=None) == call(t=2) == call(n=1 << 30) == lm.MOE_ERR_INVALID
    assert call(scale=0) == call(group=48, K=200) == lm.MOE_ERR_UNSUPPORTED and call(rows=0) == lm.MOE_ERR_INVALID


def test_the_norm_bound_sees_a_lost_plane():
    """f32 x held in one f16 per value instead of two is off by a hundred bounds, and within the bound per element."""
    rng = np.random.default_rng(1)
    K, rows, group = 2048, 400, 128
    codes = rng.integers(0, 256, size=(rows, K // 2), dtype=np.uint8)
    values, parts = R.w4_values(codes, 0.01 * (0.2 + rng.random((rows, K // group))), None, K, group)
    x = rng.normal(size=K).astype(np.float32)
    up = np.exp2(14 - np.floor(np.log2(np.abs(x).reshape(-1, 256).max(1)))).repeat(256)
    lost = (x * up).astype(np.float16).astype(np.float64) / up
    err, ref = values @ (lost - x), values @ x.astype(np.float64)
    assert np.linalg.norm(err) > 100 * R.W4_NORM * np.linalg.norm(ref)
    assert (np.abs(err) < R.w4_tol(parts @ np.abs(x), K)).all()
