"""Sorting by expert and 4-bit matrices: what is refused before anything touches a
GPU, at the C interface and in Python."""
import ctypes
from importlib import import_module

import pytest
import torch

F32, F16, BF16, Q4_0 = 0, 1, 30, 2
P = 0x1000      # an address that nothing reads


def test_sort_and_rows_refuse(pkg):
    L, lm = pkg.lib(), import_module("a6000-custom-kernels_b200._lib")
    bad, no = lm.MOE_ERR_INVALID, lm.MOE_ERR_UNSUPPORTED
    sort = lambda ids=P, stride=2, n=3, k=2, E=4, out=P: L.moe_b200_sort_by_expert(ids, stride, n, k, E, out, out, out, out, None)   # noqa: E731
    assert sort(n=-1) == bad and sort(k=0) == bad and sort(stride=1) == bad and sort(ids=None) == bad and sort(out=None) == bad
    assert sort(E=0) == no and sort(E=1025) == no and sort(n=1 << 30) == no
    for f in (lambda x=P, t=F32, s=8, n=3, k=2, H=8, o=P: L.moe_b200_gather_sorted(x, t, s, n, k, H, P, P, o, None),
              lambda x=P, t=F32, s=8, n=3, k=2, H=8, o=P: L.moe_b200_combine_sorted(x, t, s, n, k, H, P, P, None, 0, o, None),
              lambda x=P, t=F32, s=8, n=3, k=2, H=8, o=P: L.moe_b200_combine_sorted_grad(x, t, s, P, 8, n, k, H, P, P, P, o, None, None),
              lambda x=P, t=F32, s=8, n=3, k=2, H=8, o=P: L.moe_b200_dispatch_sorted(x, t, s, H, P, k, n, k, 4, P, P, P, P, o, None)):
        assert f(x=None) == bad and f(s=7) == bad and f(n=-1) == bad and f(k=0) == bad and f(H=0) == bad
        assert f(t=Q4_0) == no and f(n=1 << 30) == no
        assert f(x=P + 2) == bad and f(t=F16, x=P + 1) == bad and f(o=P + 1) == bad      # not aligned to the elements
    assert L.moe_b200_gather_sorted(None, F32, 8, 0, 2, 8, None, None, None, None) == 0
    assert L.moe_b200_combine_sorted(P, F32, 8, 3, 2, 8, P, None, P, 7, P, None) == bad
    assert L.moe_b200_combine_sorted_grad(P, F32, 8, None, 8, 3, 2, 8, P, P, P, P, P, None) == bad     # d_weights without y
    assert L.moe_b200_combine_sorted_grad(P, F32, 8, P, 8, 3, 2, 8, P, None, P, P, P, None) == bad     # d_y without their number


def _w4(lm, E=2, rows=16, K=64, group=32, scale=F16, zeros=0, data=P):
    return lm.MoeW4(data, E, rows, K, group, scale, zeros)


def test_w4_shapes(pkg):
    L, lm = pkg.lib(), import_module("a6000-custom-kernels_b200._lib")
    size = lambda **kw: L.moe_b200_w4_packed_size(ctypes.byref(_w4(lm, **kw)))   # noqa: E731
    # 16 rows x 256 values: 2048 bytes of codes, 32 (and 16) per group of them
    assert size(group=32) == 2 * (2048 + 8 * 32) and size(group=32, zeros=1) == 2 * (2048 + 8 * 48)
    assert size(group=64) == size(group=1000) == 2 * (2048 + 32)                            # one group a row
    assert size(K=300, rows=17, group=128) == 2 * 2 * 2 * (2048 + 2 * 32) and size(K=1, group=1) > 0
    assert size(K=4096, group=1024, rows=1, E=1) == 16 * (2048 + 32)
    for kw in (dict(E=0), dict(rows=0), dict(K=0), dict(group=0), dict(E=1025), dict(K=(1 << 20) + 1), dict(rows=(1 << 24) + 1),
               dict(scale=F32), dict(K=200, group=48), dict(K=200, group=16), dict(K=200, group=96)):
        assert size(**kw) == 0, kw
    ws = lambda n, k, t=F32, pp=0, **kw: L.moe_b200_w4_workspace_size(ctypes.byref(_w4(lm, **kw)), n, k, t, pp)   # noqa: E731
    assert ws(1, 8, E=8) == 0 and ws(1, 0, E=1, K=2048) == 0
    assert ws(64, 8, E=8) > 0 and ws(2000, 2, pp=1) > ws(2000, 2) > 0
    assert ws(0, 2) == ws(4, -1) == ws(4, 2, t=Q4_0) == ws(4, 2, scale=F32) == 0


def test_w4_calls_refuse(pkg):
    L, lm = pkg.lib(), import_module("a6000-custom-kernels_b200._lib")
    bad, no = lm.MOE_ERR_INVALID, lm.MOE_ERR_UNSUPPORTED

    def call(w=None, gate=None, bias=None, gate_bias=None, op=0, x=P, t=F32, stride=64, n=1, ids=P, k=2, ids_stride=2, dst=P, ws=None, b=0):
        w = _w4(lm) if w is None else w
        return L.moe_b200_w4_mul_mat_id(ctypes.byref(w), None if gate is None else ctypes.byref(gate), bias, gate_bias, op, 0.0, x, t,
                                        stride, 0, n, ids, k, ids_stride, dst, ws, b, None)
    assert L.moe_b200_w4_mul_mat_id(None, None, None, None, 0, 0.0, P, F32, 64, 0, 1, P, 2, 2, P, None, 0, None) == bad
    assert call(w=_w4(lm, data=None)) == bad and call(w=_w4(lm, data=P + 8)) == bad and call(w=_w4(lm, scale=F32)) == no
    for kw in (dict(E=3), dict(rows=17), dict(K=96), dict(group=64), dict(scale=BF16), dict(zeros=1), dict(data=None), dict(data=P + 4)):
        assert call(gate=_w4(lm, **kw)) == bad, kw
    assert call(gate_bias=P) == bad and call(gate=_w4(lm), op=5) == bad and call(gate=_w4(lm), op=-1) == bad
    assert call(t=Q4_0) == no and call(n=-1) == bad and call(k=0) == bad and call(stride=63) == bad and call(ids_stride=1) == bad
    assert call(n=1 << 30) == no and call(x=None) == bad and call(dst=None) == bad and call(x=P + 2) == bad
    assert call(ids=None) == bad and call(w=_w4(lm, E=1), ids=None, k=2) == bad                # several matrices, several picks
    assert call(n=600) == bad and b"workspace" in L.moe_b200_last_error()
    assert call(n=600, ws=P + 8, b=1 << 30) == bad and b"aligned" in L.moe_b200_last_error()
    assert call(n=0, x=None, ids=None, dst=None) == 0
    pack = lambda w, codes=P, scales=P, zeros=None, dst=P, n=1 << 20: L.moe_b200_w4_pack(ctypes.byref(w), codes, scales, zeros, dst, n, None)   # noqa: E731
    assert pack(_w4(lm), codes=None) == pack(_w4(lm), scales=None) == pack(_w4(lm), dst=None) == pack(_w4(lm), dst=P + 8) == bad
    assert pack(_w4(lm), zeros=P) == pack(_w4(lm, zeros=1)) == pack(_w4(lm), scales=P + 1) == pack(_w4(lm), n=100) == bad


def test_python_refuses_what_is_not_on_a_gpu(pkg):
    ids, x = torch.zeros((3, 2), dtype=torch.int32), torch.zeros((3, 8))
    for f in (lambda: pkg.sort_by_expert(ids, 4), lambda: pkg.dispatch_sorted(x, ids, 4), lambda: pkg.ExpertOrder(ids, 4),
              lambda: pkg.W4Weights(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.float16), 32, 32)):
        with pytest.raises(pkg.MoeError):
            f()
