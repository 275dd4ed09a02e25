"""The MXFP4 and routing entry points refuse bad arguments with a status code,
before anything touches a GPU; and the 64-bit reference's own format checks."""
import ctypes

import numpy as np
import pytest

import mx_ref as R


def _lm():
    from importlib import import_module
    return import_module("a6000-custom-kernels_b200._lib")


def test_reference_quantizer_properties():
    rng = np.random.default_rng(0)
    x = rng.normal(size=(5, 96)) * np.exp(rng.normal(size=(5, 1)) * 3)
    x[0, :32] = 0
    for planes, worst in ((1, 1 / 4), (2, 1 / 16)):
        # a plane leaves at most half a step at the top of the block: 1 of amax's [4, 8), and 2 where it saturates
        v = R.values(x, planes)
        top = np.abs(x.reshape(5, 3, 32)).max(-1).repeat(32, -1).reshape(5, 96)
        assert (np.abs(v - x) <= worst * top).all()
    assert (R.values(x, 1)[0, :32] == 0).all()
    b = R.quantize(R.values(x, 1), 1)[0]           # values on the grid keep their values
    assert np.array_equal(R.from_blocks(b, 96), R.values(x, 1))


def test_reference_matches_the_format_of_gguf():
    """Block decoding against gguf-py's MXFP4, where this machine has it."""
    quants = pytest.importorskip("gguf.quants")
    gguf = pytest.importorskip("gguf")
    if not hasattr(gguf.GGMLQuantizationType, "MXFP4"):
        pytest.skip("gguf without MXFP4")
    rng = np.random.default_rng(1)
    blocks = rng.integers(0, 256, size=(64, 17), dtype=np.uint8)
    blocks[:, 0] = rng.integers(100, 150, size=64)
    want = quants.dequantize(blocks.reshape(1, -1), gguf.GGMLQuantizationType.MXFP4).reshape(64, 32)
    assert np.array_equal(R.from_blocks(blocks, 32).astype(np.float32), want)


def test_packed_size(pkg):
    L = pkg.lib()
    assert L.moe_b200_mxfp4_packed_size(3, 100, 96) == 3 * 8704
    assert L.moe_b200_mxfp4_packed_size(2, 129, 160) == 2 * 2 * 2 * 8704
    for bad in ((0, 128, 128), (1, 0, 128), (1, 128, 0), (1, 128, 48), (5000, 128, 128)):
        assert L.moe_b200_mxfp4_packed_size(*bad) == 0


def test_struct_layouts(pkg):
    lm = _lm()
    assert ctypes.sizeof(lm.MoeRouter) == 24
    assert ctypes.sizeof(lm.MoeMxfp4) == 32
    assert ctypes.sizeof(lm.MoeMxfp4Layer) == 6 * 32 + 3 * 8 + 8 + 12 + 24 + 4 + 8


@pytest.mark.parametrize("kw, code", [
    (dict(x_type=3), "UNSUPPORTED"), (dict(cols=48), "INVALID"), (dict(cols=0), "INVALID"), (dict(rows=-1), "INVALID"),
    (dict(stride=32), "INVALID"), (dict(planes=0), "INVALID"), (dict(planes=3), "INVALID"), (dict(x=None), "INVALID"),
    (dict(x=0x1002), "INVALID"), (dict(rows=1 << 60), "INVALID"),
])
def test_quantize_refusals(pkg, kw, code):
    lm = _lm()
    a = dict(x=0x1000, x_type=0, rows=4, cols=64, stride=64, planes=1)
    a.update(kw)
    want = getattr(lm, "MOE_ERR_" + code)
    L = pkg.lib()
    assert L.moe_b200_quantize_mxfp4(a["x"], a["x_type"], a["rows"], a["cols"], a["stride"], a["planes"], 0x2000, None) == want
    assert L.moe_b200_dequantize_mxfp4(0x2000, a["rows"], a["cols"], a["planes"], a["x"], a["x_type"], a["stride"], None) == want


@pytest.mark.parametrize("kw, code", [
    (dict(n_experts=0), "UNSUPPORTED"), (dict(n_experts=1025), "UNSUPPORTED"), (dict(k=0), "INVALID"), (dict(k=33), "INVALID"),
    (dict(k=9, n_group=8, topk_group=1), "INVALID"), (dict(n_group=3), "INVALID"), (dict(n_group=0), "INVALID"),
    (dict(n_group=64), "INVALID"), (dict(topk_group=2), "INVALID"), (dict(score=3), "INVALID"), (dict(group_score=2), "INVALID"),
    (dict(dtype=2), "UNSUPPORTED"), (dict(stride=63), "INVALID"), (dict(n_tok=-1), "INVALID"), (dict(logits=None), "INVALID"),
    (dict(logits=0x1001), "INVALID"),
])
def test_route_refusals(pkg, kw, code):
    lm = _lm()
    a = dict(logits=0x1000, dtype=0, stride=64, n_tok=2, n_experts=64, k=8, score=0, n_group=1, topk_group=1, group_score=0)
    a.update(kw)
    r = lm.MoeRouter(a["score"], a["n_group"], a["topk_group"], a["group_score"], 0, 1.0)
    rc = pkg.lib().moe_b200_route_experts(ctypes.byref(r), a["logits"], a["dtype"], max(a["stride"], a["n_experts"]) if "stride" not in kw else a["stride"],
                                          None, a["n_tok"], a["n_experts"], a["k"], 0x2000, 0x3000, None)
    assert rc == getattr(lm, "MOE_ERR_" + code)


def test_route_and_product_of_no_tokens(pkg):
    lm = _lm()
    r = lm.MoeRouter(0, 1, 1, 0, 0, 1.0)
    assert pkg.lib().moe_b200_route_experts(ctypes.byref(r), None, 0, 64, None, 0, 64, 8, None, None, None) == lm.MOE_OK
    w = lm.MoeMxfp4(0x1000, 4, 128, 128)
    assert pkg.lib().moe_b200_mxfp4_mul_mat_id(ctypes.byref(w), None, None, None, 0, 0.0, None, 0, 128, 0, 0, None, 2, 2, 2, None,
                                               None, 0, None) == lm.MOE_OK


@pytest.mark.parametrize("kw, code", [
    (dict(data=None), "INVALID"), (dict(data=0x1008), "INVALID"), (dict(K=100), "INVALID"), (dict(rows=0), "INVALID"),
    (dict(E=4097), "UNSUPPORTED"), (dict(gate=(0x1000, 4, 128, 64)), "INVALID"), (dict(gate_bias=0x1000), "INVALID"),
    (dict(gate=(0x1000, 4, 128, 128), glu=9), "INVALID"), (dict(x_type=10), "UNSUPPORTED"), (dict(planes=3), "INVALID"),
    (dict(k=0), "INVALID"), (dict(ids_stride=1), "INVALID"), (dict(x_stride=96), "INVALID"), (dict(n_tok=1 << 40), "UNSUPPORTED"),
    (dict(x=None), "INVALID"), (dict(n_tok=33, ws_bytes=100), "INVALID"), (dict(n_tok=40, k=2, ws=None), "INVALID"),
    (dict(ws=0x1004), "INVALID"),
])
def test_product_refusals(pkg, kw, code):
    lm = _lm()
    a = dict(data=0x1000, E=4, rows=128, K=128, gate=None, gate_bias=None, glu=0, x=0x1000, x_type=0, x_stride=128, n_tok=3, k=2,
             ids_stride=2, planes=2, ws=0x1000, ws_bytes=1 << 30)
    a.update(kw)
    w = lm.MoeMxfp4(a["data"], a["E"], a["rows"], a["K"])
    g = lm.MoeMxfp4(*a["gate"]) if a["gate"] else None
    rc = pkg.lib().moe_b200_mxfp4_mul_mat_id(ctypes.byref(w), ctypes.byref(g) if g else None, None, a["gate_bias"], a["glu"], 0.0,
                                             a["x"], a["x_type"], a["x_stride"], 0, a["n_tok"], 0x1000, a["k"], a["ids_stride"],
                                             a["planes"], 0x1000, a["ws"], a["ws_bytes"], None)
    assert rc == getattr(lm, "MOE_ERR_" + code), pkg.lib().moe_b200_last_error()


def test_workspace_grows_with_the_call(pkg):
    lm = _lm()
    w = lm.MoeMxfp4(0x1000, 16, 256, 512)
    size = pkg.lib().moe_b200_mxfp4_workspace_size
    assert 0 < size(ctypes.byref(w), 17, 4, 1) < size(ctypes.byref(w), 17, 4, 2) < size(ctypes.byref(w), 300, 4, 2)
    assert size(ctypes.byref(w), 16, 4, 2) == 0 < size(ctypes.byref(w), 13, 5, 2)     # a few tokens need none
    assert size(ctypes.byref(w), 1, 0, 1) == 0 and size(ctypes.byref(w), 1, 4, 3) == 0 and size(None, 1, 4, 1) == 0


def test_layer_refusals(pkg):
    lm = _lm()
    L = pkg.lib()

    def desc(F=256, H=512, E=8, k=2, **kw):
        d = lm.MoeMxfp4Layer()
        d.gate, d.up, d.down = (lm.MoeMxfp4(0x1000, E, F, H), lm.MoeMxfp4(0x1000, E, F, H), lm.MoeMxfp4(0x1000, E, H, F))
        d.k, d.planes, d.router = k, 2, lm.MoeRouter(0, 1, 1, 0, 0, 1.0)
        for n, v in kw.items():
            setattr(d, n, v)
        return d

    assert L.moe_b200_mxfp4_layer_workspace_size(ctypes.byref(desc()), 3) > 0
    for d in (desc(k=0), desc(k=9), desc(planes=3), desc(gate=lm.MoeMxfp4(0x1000, 8, 128, 512)),
              desc(down=lm.MoeMxfp4(0x1000, 8, 512, 512)), desc(shared_up=lm.MoeMxfp4(0x1000, 1, 256, 512))):
        assert L.moe_b200_mxfp4_layer_workspace_size(ctypes.byref(d), 3) == 0
        assert L.moe_b200_mxfp4_layer_run(ctypes.byref(d), 0x1000, 0, 512, 0x1000, 0, 8, 0x1000, 3, 0x1000, 1 << 30,
                                          None) == lm.MOE_ERR_INVALID
    assert L.moe_b200_mxfp4_layer_run(ctypes.byref(desc()), 0x1000, 0, 512, 0x1000, 0, 8, 0x1000, 3, 0x1000, 64,
                                      None) == lm.MOE_ERR_INVALID


def test_python_refusals_without_a_gpu(pkg):
    import torch
    x = torch.zeros((2, 64))
    for call in (lambda: pkg.quantize_mxfp4(x), lambda: pkg.dequantize_mxfp4(torch.zeros((2, 34), dtype=torch.uint8), 64),
                 lambda: pkg.MXFP4Weights(torch.zeros((2, 4, 34), dtype=torch.uint8), 64, 4), lambda: pkg.route_experts(x, 2),
                 lambda: pkg.Router(2, score="relu"), lambda: pkg.Router(2, group_score="sum"),
                 lambda: pkg.Router(2, bias=torch.zeros(64)),
                 lambda: pkg.MoELayer(64, 64, 4, 2, {"gate": pkg.moe_cache.MXFP4, "up": 2, "down": 2}),
                 lambda: pkg.MoELayer(64, 64, 4, 2, {r: pkg.moe_cache.MXFP4 for r in ("gate", "up", "down")}, host=True)):
        with pytest.raises(pkg.MoeError):
            call()


def test_a_layer_with_its_own_router_stays_off_paths_that_route_themselves(pkg):
    from importlib import import_module
    from types import SimpleNamespace
    ep = import_module("a6000-custom-kernels_b200.ep")
    layer = SimpleNamespace(router=object())
    with pytest.raises(pkg.MoeError, match="router"):
        pkg.Stack([SimpleNamespace(router=None), layer], [], [], [])
    with pytest.raises(pkg.MoeError, match="router"):
        ep.EPMoELayer(layer, 0, 2)


def test_layer_arguments_by_position(pkg):
    """`shared` and what follows may be given by position, for every type."""
    mc = pkg.moe_cache
    assert type(pkg.MoELayer.__new__(pkg.MoELayer, 64, 64, 4, 2, {r: mc.Q4_0 for r in ("gate", "up", "down")}, False)) is pkg.MoELayer
    with pytest.raises(pkg.MoeError, match="device memory"):
        pkg.MoELayer(64, 64, 4, 2, {r: mc.MXFP4 for r in ("gate", "up", "down")}, False, host=True)
