"""Layers with a router of their own: what they keep between calls, and what
they answer about them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

MX = 39


@pytest.fixture(params=[MX, 2], ids=["mxfp4", "q4_0"])
def layer(request, pkg, cuda):
    pkg.moe_cache.configure(enabled=True)
    types = {r: request.param for r in ("gate", "up", "down")}
    yield pkg.MoELayer(256, 128, 8, 2, types, device=cuda, seed=3, router=pkg.Router(2, "sigmoid", norm_w=True))
    pkg.moe_cache.reset()


def _tokens(n, cuda, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randn((n, 256), generator=g, device=cuda), torch.randn((n, 8), generator=g, device=cuda)


def test_lengths_leave_no_memory_behind(pkg, cuda, layer):
    """Prompts of many lengths: what the layer keeps is one call's, not one per length."""
    x, lg = _tokens(512, cuda)
    layer.prefill(x, lg)
    torch.cuda.synchronize()
    kept = torch.cuda.memory_allocated()
    for n in range(100, 500, 40):
        layer.prefill(x[:n], lg[:n])
    layer.prefill(x, lg)
    assert torch.cuda.memory_allocated() <= kept
    small = torch.cuda.memory_allocated()
    layer.decode(x[:1], lg[:1])
    assert torch.cuda.memory_allocated() < small


def test_calls_of_one_length_side_by_side(pkg, cuda, layer):
    """Eager calls on two streams at once, and two captured ones replayed at once while eager calls of other
    lengths come and go: each call has a workspace of its own."""
    n = 96
    data = [_tokens(n, cuda, seed) for seed in (1, 2)]
    alone = [layer.prefill(x, lg).clone() for x, lg in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(10):
        got = [layer.prefill(x, lg, stream=s) for (x, lg), s in zip(data, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))
    graphs, outs = [], []
    for x, lg in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.prefill(x, lg))
        graphs.append(g)
    big = _tokens(400, cuda, 3)
    want = layer.prefill(*big).clone()
    for i in range(10):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        assert torch.equal(layer.prefill(*big), want)
        layer.prefill(big[0][: 97 + i], big[1][: 97 + i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, alone))
    assert pkg.moe_cache.device_error() == 0


def test_what_a_routed_layer_says_of_its_last_call(pkg, cuda, layer):
    """One launch is what the layer without a router makes; the last call's routing is its own; parts that the
    call does not keep, or that another call has replaced, are refused."""
    assert not layer.fused(1)
    with pytest.raises(pkg.MoeError):
        layer.routing_of(5)
    x, lg = _tokens(5, cuda)
    layer.decode(x, lg)
    ids, w = layer.routing_of(5)
    i, v = layer.router(lg)
    assert torch.equal(ids, i) and torch.equal(w, v)
    layer.prefill(*_tokens(7, cuda, 1))
    assert layer.routing_of(7)[0].shape == (7, 2)
    for call in (layer.routing_of, layer.intermediates, layer.prefill_intermediates):
        with pytest.raises(pkg.MoeError):
            call(5)
    with pytest.raises(pkg.MoeError):
        layer.prefill_intermediates(7)


def test_tensors_of_another_device_are_refused(pkg, cuda, layer):
    """The experts lie on the layer's device: tokens of another one are refused (here the layer is told that it
    lives elsewhere)."""
    x, lg = _tokens(2, cuda)
    layer.decode(x, lg)
    layer.device = torch.device("cuda", 1)
    with pytest.raises(pkg.MoeError, match="device"):
        layer.decode(x, lg)
