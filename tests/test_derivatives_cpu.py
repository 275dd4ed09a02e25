"""Calls that have no derivative, or none of a kind, say so: what of that needs no GPU."""
from importlib import import_module

import pytest
import torch
from torch.autograd import forward_ad


def test_tangents_are_refused(pkg):
    call = import_module("a6000-custom-kernels_b200._call")
    x = torch.ones(3)
    call.no_tangents(x, None)
    with forward_ad.dual_level():
        call.no_tangents(x, None)
        dual = forward_ad.make_dual(x, torch.ones(3))
        for t in (dual, dual * 2):
            with pytest.raises(pkg.MoeError, match="forward"):
                call.no_tangents(x, None, t)
    call.no_tangents(x, None)


def test_a_product_of_4_bit_matrices_keeps_its_place_in_a_graph(pkg):
    w4 = import_module("a6000-custom-kernels_b200.w4")
    x, plain = torch.ones(3, requires_grad=True), torch.ones(3)
    assert w4._wants_grad(None, x, None) and w4._wants_grad(None, plain, None, x) and not w4._wants_grad(plain, plain, None)
    with torch.no_grad():
        assert not w4._wants_grad(None, x) and not w4._wants_grad(plain, x)
    with pytest.raises(pkg.MoeError, match="dst"):
        w4._wants_grad(plain, x)
    y = w4._NoGradient.apply(torch.full, ((2,), 5.0), x, None, plain)
    assert y.requires_grad and y.tolist() == [5.0, 5.0]
    with pytest.raises(pkg.MoeError, match="no gradient"):
        y.sum().backward()
    assert x.grad is None


class _Made(torch.autograd.Function):
    """Stands for the calls' autograd nodes."""
    @staticmethod
    def forward(ctx, t, made):
        ctx.made = made
        import_module("a6000-custom-kernels_b200.sorted")._remember(ctx)
        return t * 2

    @staticmethod
    def backward(ctx, g):
        return 2 * g, None


def test_captures_next_to_graphs_of_the_same_leaves(pkg, monkeypatch):
    """Whether the leaves themselves are taken or what other operations made of them, on either side."""
    check = import_module("a6000-custom-kernels_b200.sorted")._check_capture
    p, q = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    for first in (lambda: _Made.apply(p, 7), lambda: _Made.apply(p * 3, 7).sum(), lambda: _Made.apply(p + torch.ones(3) @ torch.ones(3), 7)):
        kept = first()
        for of in (lambda: p, lambda: p.sin(), lambda: (p + q).exp(), lambda: _Made.apply(p * 5, 7)):
            now = of()
            monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            for args in ((now,), (None, q, now)):
                with pytest.raises(pkg.MoeError, match="alive"):
                    check(8, *args)
            check(7, now)                                     # (the stream of the kept graph)
            check(8, q, q.cos(), None, torch.ones(3), p.detach())
            monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
            check(8, now)
            del now, args
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        del kept
        check(8, p, p.sin())
