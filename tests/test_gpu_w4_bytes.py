"""Laid-out 4-bit matrices whose bytes another kernel has written: products come behind it."""
from importlib import import_module

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(pkg, cuda, seed, E=None, rows=4096, K=4096, group=128):
    g = torch.Generator(device=cuda).manual_seed(seed)
    shape = (rows,) if E is None else (E, rows)
    codes = torch.randint(0, 256, (*shape, K // 2), generator=g, device=cuda, dtype=torch.uint8)
    scales = (0.01 * torch.rand((*shape, K // group), generator=g, device=cuda)).half()
    return pkg.W4Weights(codes, scales, K, group)


class Calls:
    """The library, with the names of the functions that were called."""
    def __init__(self, lib):
        self.lib, self.names = lib, []

    def __getattr__(self, name):
        self.names.append(name)
        return getattr(self.lib, name)

    def took(self):
        names, self.names = [n for n in self.names if "size" not in n], []
        return [n.removeprefix("moe_b200_w4_") for n in names]


def test_which_products_settle(pkg, cuda, monkeypatch):
    w, gate, experts = make(pkg, cuda, 1, rows=64, K=256), make(pkg, cuda, 2, rows=64, K=256), make(pkg, cuda, 3, E=2, rows=64, K=256)
    x, ids = torch.randn((3, 256), device=cuda), torch.zeros((3, 1), dtype=torch.int32, device=cuda)
    calls = Calls(pkg.lib())
    monkeypatch.setattr(import_module("a6000-custom-kernels_b200.w4"), "lib", lambda: calls)
    pkg.w4_mul_mat(w, x, gate=gate)
    pkg.w4_mul_mat_id(experts, x, ids)
    assert calls.took() == ["mul_mat_id"] * 2
    assert gate.data.dtype == experts.data.dtype == torch.uint8
    for _ in range(2):
        pkg.w4_mul_mat(w, x, gate=gate)
        pkg.w4_mul_mat_id(experts, x, ids)
        pkg.w4_mul_mat(w, x)
        assert calls.took() == ["settle", "mul_mat_id"] * 2 + ["mul_mat_id"]
    gate.settle()
    experts.settle(torch.cuda.Stream())
    pkg.w4_mul_mat(w, x, gate=gate)
    pkg.w4_mul_mat_id(experts, x, ids)
    assert calls.took() == ["settle"] * 2 + ["mul_mat_id"] * 2


@pytest.mark.parametrize("settled", [False, True])
def test_products_right_behind_a_kernel_that_writes_the_bytes(pkg, cuda, settled):
    ws = [make(pkg, cuda, s) for s in (1, 2)]
    xs = [torch.randn((n, 4096), device=cuda, dtype=torch.float16) for n in (1, 24)]     # 24: x is staged by a launch between
    want = [[pkg.w4_mul_mat(w, x) for x in (*xs, *xs[::-1])] for w in ws]
    assert not torch.equal(want[0][0], want[1][0])
    to = make(pkg, cuda, 3)
    sources = [w.data ^ 0x5A for w in ws]
    torch.cuda.synchronize()

    def run():
        got = []
        for src in sources:
            torch.bitwise_xor(src, 0x5A, out=to.data)        # a kernel that the library knows nothing of
            if settled:
                to.settle()
            got.append([pkg.w4_mul_mat(to, x) for x in (*xs, *xs[::-1])])
        return got
    for _ in range(5):
        got = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(want, got) for a, b in zip(p, q))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for p, q in zip(want, got) for a, b in zip(p, q))
    assert pkg.moe_cache.device_error() == 0
