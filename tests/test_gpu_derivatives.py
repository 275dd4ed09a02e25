"""Products with 4-bit matrices have no derivatives, the sorted rows none in forward mode: both say so where one is asked for."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture()
def matrices(pkg, cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    codes = torch.randint(0, 256, (3, 24, 32), generator=g, device=cuda, dtype=torch.uint8)
    scales = torch.rand((3, 24, 2), generator=g, device=cuda).half()
    return pkg.W4Weights(codes, scales, 64, 32), pkg.W4Weights(codes[0], scales[0], 64, 32)


def test_products_of_inputs_that_require_gradients(pkg, cuda, matrices):
    w, one = matrices
    x = torch.randn((5, 64), device=cuda)
    ids = torch.from_numpy(np.arange(10, dtype=np.int32).reshape(5, 2) % 3).to(cuda)
    b, b1 = torch.randn((3, 24), device=cuda), torch.randn((1, 24), device=cuda)
    calls = [lambda x, b, b1, **kw: pkg.w4_mul_mat(one, x, bias=b1, **kw),
             lambda x, b, b1, **kw: pkg.w4_mul_mat(one, x, gate=one, bias=b1, gate_bias=b1, **kw),
             lambda x, b, b1, **kw: pkg.w4_mul_mat_id(w, x, ids, bias=b, **kw),
             lambda x, b, b1, **kw: pkg.w4_mul_mat_id(w, x, ids, gate=w, bias=b, gate_bias=b, stream=torch.cuda.Stream(), **kw)]
    for call in calls:
        torch.cuda.synchronize()
        want = call(x, b, b1)
        assert not want.requires_grad
        for grads in ((True, False), (False, True), (True, True)):
            xl, bl, bl1 = (t.detach().clone().requires_grad_(on) for t, on in zip((x, b, b1), (grads[0], grads[1], grads[1])))
            torch.cuda.synchronize()
            got = call(xl, bl, bl1)
            torch.cuda.synchronize()
            assert got.requires_grad and torch.equal(got.detach(), want)
            with pytest.raises(pkg.MoeError, match="no gradient"):
                got.sum().backward()
            with pytest.raises(pkg.MoeError, match="dst"):
                call(xl, bl, bl1, dst=torch.empty_like(want))
            with torch.no_grad():
                dst = torch.empty_like(want)
                plain = call(xl, bl, bl1)
                assert call(xl, bl, bl1, dst=dst) is dst and not plain.requires_grad
                torch.cuda.synchronize()
                assert torch.equal(dst, want) and torch.equal(plain, want)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: calls[0](dual, b, b1), lambda: calls[2](dual, b, b1),
                  lambda: calls[0](x, b, forward_ad.make_dual(b1, b1))):
            with pytest.raises(pkg.MoeError, match="forward"):
                f()
        assert torch.equal(calls[0](x, b, b1), pkg.w4_mul_mat(one, x, bias=b1))


def test_the_chain_around_a_product_trains_up_to_it_only(pkg, cuda, matrices):
    """dispatch, product, combine: the weights have a gradient, the tokens' is refused."""
    w, _ = matrices
    x = torch.randn((6, 64), device=cuda, requires_grad=True)
    ids = torch.from_numpy(np.arange(12, dtype=np.int32).reshape(6, 2) % 3).to(cuda)
    weights = torch.rand((6, 2), device=cuda, requires_grad=True)
    for of in (x, x.detach()):
        rows, order = pkg.dispatch_sorted(of, ids, 3)
        y = pkg.w4_mul_mat_id(w, rows, order.experts.view(-1, 1))[:, 0]
        out = pkg.combine_sorted(y, order, weights)
        if of is x:
            with pytest.raises(pkg.MoeError, match="no gradient"):
                out.sum().backward()
        else:
            weights.grad = None
            out.sum().backward()
    # sums of 24 values in 32 bits: 23 additions
    y, at = y.detach().double(), order.positions.long()
    assert ((weights.grad.double() - y.sum(1)[at]).abs() <= 24 * 2.0 ** -24 * y.abs().sum(1)[at]).all() and x.grad is None


def test_forward_mode_through_sorted_rows(pkg, cuda):
    ids = torch.from_numpy(np.arange(12, dtype=np.int32).reshape(6, 2) % 3).to(cuda)
    x, y, w = torch.randn((6, 40), device=cuda), torch.randn((12, 40), device=cuda), torch.rand((6, 2), device=cuda)
    order = pkg.sort_by_expert(ids, 3)
    with forward_ad.dual_level():
        for grad in (False, True):
            dx, dy, dw = (forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t)) for t in (x, y, w))
            for f in (lambda: pkg.dispatch_sorted(dx, ids, 3), lambda: pkg.gather_sorted(dx, order),
                      lambda: pkg.combine_sorted(dy, order, w), lambda: pkg.combine_sorted(y, order, dw),
                      lambda: pkg.combine_sorted(y, order, w, shared=dx)):
                with pytest.raises(pkg.MoeError, match="forward"):
                    f()
        assert torch.equal(pkg.dispatch_sorted(x, ids, 3)[0], pkg.gather_sorted(x, order))
    # (torch.func's wrappers have no memory of their own: torch refuses them)
    with pytest.raises(Exception):
        torch.func.jvp(lambda t: pkg.gather_sorted(t, order), (x,), (torch.ones_like(x),))


def test_capture_next_to_an_eager_graph_of_what_leaves_became(pkg, cuda):
    """The calls take no leaf but what another operation made of it: refused next to a live graph of the same leaf."""
    ids = torch.from_numpy(np.arange(12, dtype=np.int32).reshape(6, 2) % 3).to(cuda)
    p, d = torch.randn((6, 40), device=cuda, requires_grad=True), torch.randn((12, 40), device=cuda)
    side = torch.cuda.Stream()

    def step():
        rows, order = pkg.dispatch_sorted(p * 2, ids, 3)
        return rows, torch.autograd.grad(rows, p, d)[0], order
    alive = step()
    want = alive[1].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        with pytest.raises(pkg.MoeError, match="alive"):
            pkg.dispatch_sorted(p * 2, ids, 3)
        with pytest.raises(pkg.MoeError, match="alive"):
            pkg.gather_sorted(p, alive[2])
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        _, got, _ = step()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
