"""One MoE FFN layer on the B200 path: the graph around two MUL_MAT_ID calls.

Routing (top-k + softmax), the fused gate/up GEMV with the GLU and the shared
expert, the down GEMV and the weighted combine run as four sm_100a launches of
libmoe_b200.so (moe_b200_layer_decode). This mirrors what llama.cpp's graph does
around the reference's intercepted MUL_MAT_ID calls (build_moe_ffn order:
route, gate/up, GLU, down, weight, sum over picks, add the shared expert).
"""
import ctypes
import math

import torch

from ._call import ELEM, bad, dense_rows, given, keep, on
from ._lib import MoeLayerDesc, MoeMxfp4Layer, check, lib
from .moe_cache import GLU_SWIGLU, MXFP4, _ptr, _stream, expert_tensor, fill_quantized, row_size
from .mxfp4 import MXFP4Weights, quantize_mxfp4
from .router import Router


def _checked_router(router, k, norm_w):
    if router is not None:
        if router.k != k:
            raise bad("the router picks another number of experts than the layer has")
        if norm_w and not router.desc.norm_w:
            raise bad("norm_w with a router that does not normalise: the layer takes the router's weights (Router(norm_w=True))")
    return router


class MoELayer:
    """Expert weights live in `device` memory (HBM-resident) unless `host=True`,
    in which case they live in pinned host memory behind the tiered cache.

    `router` (a Router) makes tokens pick their experts as it says, through
    decode and prefill alike; None is softmax over all experts, top-k. A router
    brings its own norm_w: the layer's may repeat it, not contradict it.
    MoELayer(..., types with MXFP4 for gate, up and down) makes an MXFP4Layer."""

    def __new__(cls, H=None, F=None, n_experts=None, k=None, types=None, *args, **kw):
        if cls is MoELayer and types is not None and MXFP4 in dict(types).values():
            return super().__new__(MXFP4Layer)
        return super().__new__(cls)

    def __init__(self, H, F, n_experts, k, types, shared=True, glu_op=GLU_SWIGLU, glu_limit=0.0, norm_w=False,
                 device="cuda", host=False, name="blk.0", seed=0, weights=None, sigma=0.02, router=None):
        self.H, self.F, self.E, self.k = H, F, n_experts, k
        self.router = _checked_router(router, k, norm_w)
        self.types = dict(types)          # {"gate": t, "up": t, "down": t}
        self.glu_op, self.glu_limit, self.norm_w = glu_op, glu_limit, norm_w
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device(self.device.type, torch.cuda.current_device())
        shapes = {"gate": (F, H), "up": (F, H), "down": (H, F)}
        self.w = {}
        for i, role in enumerate(("gate", "up", "down")):
            t = self.types[role]
            rows, K = shapes[role]
            if weights is not None:
                src = torch.as_tensor(weights[role])
                buf = src.pin_memory() if host else src.to(self.device)
            else:
                buf = torch.empty((n_experts, rows, row_size(t, K)), dtype=torch.uint8, device=self.device)
                fill_quantized(t, buf, n_experts * rows, K, seed * 1000003 + i, sigma=sigma)
                if host:
                    pinned = torch.empty(buf.shape, dtype=torch.uint8, pin_memory=True)
                    pinned.copy_(buf)
                    buf = pinned
            self.w[role] = buf
        self.desc_t = {r: expert_tensor(self.w[r], self.types[r], shapes[r][1], shapes[r][0],
                                        name=f"{name}.ffn_{r}_exps.weight") for r in ("gate", "up", "down")}
        self.shared = {}
        if shared:
            for i, role in enumerate(("gate", "up", "down")):
                t = self.types[role]
                rows, K = shapes[role]
                if weights is not None and weights.get(f"shared_{role}") is not None:
                    buf = torch.as_tensor(weights[f"shared_{role}"]).to(self.device)
                else:
                    buf = torch.empty((rows, row_size(t, K)), dtype=torch.uint8, device=self.device)
                    fill_quantized(t, buf, rows, K, seed * 1000003 + 7 + i, sigma=sigma)
                self.shared[role] = buf
        d = MoeLayerDesc()
        d.gate, d.up, d.down = self.desc_t["gate"], self.desc_t["up"], self.desc_t["down"]
        d.shared_type = self.types["up"] if shared else -1
        d.shared_gate = _ptr(self.shared.get("gate"))
        d.shared_up = _ptr(self.shared.get("up"))
        d.shared_down = _ptr(self.shared.get("down"))
        d.H, d.F, d.n_experts, d.k = H, F, n_experts, k
        d.glu_op, d.glu_limit, d.norm_w = glu_op, glu_limit, int(norm_w)
        self.desc = d
        self._ws, self._routed_key = {}, None

    def weight_bytes_per_token(self):
        """Expert bytes one batch-1 token streams: k routed + shared experts x 3 matrices."""
        per = sum(self.w[r][0].numel() for r in ("gate", "up", "down"))
        return per * (self.k + (1 if self.shared else 0))

    def workspace(self, n_tok):
        ws = self._ws.get(n_tok)
        if ws is None:
            nbytes = lib().moe_b200_layer_workspace_size(ctypes.byref(self.desc), n_tok)
            # zero-filled once: the fused kernel's launch epoch lives at its start
            ws = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
            self._ws[n_tok] = ws
        return ws

    def fused(self, n_tok):
        """True when decode() runs the layer as one fused kernel for n_tok tokens."""
        if self.router is not None:      # decode() runs the prefill's calls
            return False
        return bool(lib().moe_b200_layer_fused(ctypes.byref(self.desc), n_tok))

    def decode(self, x, logits, out=None, stream=None, trace=None):
        """x f32 [n_tok, H], logits f32 [n_tok, E] (device) -> out f32 [n_tok, H].
        With `trace` (a seed.TraceWriter) the step's routing is appended as one
        record per expert tensor, as the reference's trace hook writes it for
        each MUL_MAT_ID (this reads the ids back to the host)."""
        n_tok = x.shape[0]
        if self.router is not None:
            return self._routed(x, logits, out, stream, trace)
        if out is None:
            out = torch.empty((n_tok, self.H), dtype=torch.float32, device=self.device)
        ws = self.workspace(n_tok)
        check(lib().moe_b200_layer_decode(ctypes.byref(self.desc), _ptr(x), _ptr(logits), _ptr(out), n_tok,
                                          _ptr(ws), ws.numel(), _stream(stream)))
        if trace is not None:
            ids = self.routing_of(n_tok)[0].cpu().numpy()
            for r in ("gate", "up", "down"):
                trace.record(self.desc_t[r].name.decode(), ids, self.E)
        return out

    def prefill(self, x, logits, out=None, stream=None):
        """x f32 [n_tok, H], logits f32 [n_tok, E] (device) -> out f32 [n_tok, H] for any
        n_tok: the tensor-core prefill path (moe_b200_layer_prefill)."""
        n_tok = x.shape[0]
        if self.router is not None:
            return self._routed(x, logits, out, stream)
        if out is None:
            out = torch.empty((n_tok, self.H), dtype=torch.float32, device=self.device)
        key = ("prefill", n_tok)
        ws = self._ws.get(key)
        if ws is None:
            nbytes = lib().moe_b200_layer_prefill_workspace_size(ctypes.byref(self.desc), n_tok)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            self._ws[key] = ws
        check(lib().moe_b200_layer_prefill(ctypes.byref(self.desc), _ptr(x), _ptr(logits), _ptr(out), n_tok,
                                           _ptr(ws), ws.numel(), _stream(stream)))
        return out

    def _routed(self, x, logits, out, stream, trace=None):
        """The layer with its own router: route, the experts of the picks, the
        shared expert, combine (any n_tok >= 1; x contiguous f32). Every call has buffers
        of its own, allocated on its stream; the layer keeps the last call's."""
        n_tok, dev = x.shape[0], self.device
        if x.dtype != torch.float32 or x.device != dev or not x.is_contiguous() or tuple(x.shape) != (n_tok, self.H) or \
                n_tok < 1 or tuple(logits.shape) != (n_tok, self.E) or logits.device != dev:
            raise bad("x must be contiguous f32 [n_tok, H] with n_tok >= 1 and logits [n_tok, n_experts], on the layer's device")
        ctx, st = on(dev, stream)
        with ctx:
            out = torch.empty((n_tok, self.H), dtype=torch.float32, device=dev) if out is None else \
                given(out, "out", torch.float32, (n_tok, self.H), dev)
            ids, w = self.router(logits)
            self._ws.pop(self._routed_key, None)
            nbytes = lib().moe_b200_experts_prefill_workspace_size(ctypes.byref(self.desc), n_tok, self.k)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            y = torch.empty((n_tok, self.k, self.H), dtype=torch.float32, device=dev)
            ys = torch.empty((n_tok, self.H), dtype=torch.float32, device=dev) if self.shared else None
            self._routed_key = ("routed", n_tok)
            self._ws[self._routed_key] = ws, y, ys, ids, w
            check(lib().moe_b200_experts_prefill(ctypes.byref(self.desc), _ptr(x), 0, _ptr(ids), n_tok, self.k, _ptr(y),
                                                 _ptr(ws), ws.numel(), st))
            if ys is not None:
                check(lib().moe_b200_shared_prefill(ctypes.byref(self.desc), _ptr(x), n_tok, _ptr(ys), _ptr(ws), ws.numel(), st))
            check(lib().moe_b200_combine(_ptr(y), _ptr(w), _ptr(ys), _ptr(out), n_tok, self.H, self.k, st))
            picks = None if trace is None else ids.cpu().numpy()   # (waits for the stream that wrote them)
        if stream is not None:
            keep(stream, x, logits, out, self.router.bias, *self.shared.values(), *(b for b in self.w.values() if b.is_cuda))
        if trace is not None:
            for r in ("gate", "up", "down"):
                trace.record(self.desc_t[r].name.decode(), picks, self.E)
        return out

    def prefill_intermediates(self, n_tok):
        """Views of the last prefill's workspace (layout of moe_b200_layer_prefill):
        ids [n][k], weights [n][k], gate [n][k][F], h [n][k][F] (GLU output),
        y [n][k][H] (down outputs), then with a shared expert its gate [n][F],
        hs [n][F] and ys [n][H]. Refused for a layer with a router, which lays its
        calls out differently (routing_of)."""
        self._routes_itself()
        ws = self._ws[("prefill", n_tok)]
        n, k, F, H = n_tok, self.k, self.F, self.H
        parts = [(n * k, torch.int32, (n, k)), (n * k, torch.float32, (n, k)), (n * k * F, torch.float32, (n, k, F)),
                 (n * k * F, torch.float32, (n, k, F)), (n * k * H, torch.float32, (n, k, H))]
        if self.shared:
            parts += [(n * F, torch.float32, (n, F)), (n * F, torch.float32, (n, F)), (n * H, torch.float32, (n, H))]
        out, off = [], 0
        for count, dt, shape in parts:
            nbytes = 4 * count
            out.append(ws[off: off + nbytes].view(dt).view(shape))
            off += (nbytes + 255) // 256 * 256
        return tuple(out)

    def intermediates(self, n_tok):
        """Views of the last decode's workspace (layout of moe_b200_layer_decode):
        ids [n][k], weights [n][k], h [n][k][F] (GLU output), hs [n][F] (shared
        GLU output), y [n][k][H] (down outputs), ys [n][H] (shared down). Refused for a
        layer with a router, which lays its calls out differently (routing_of)."""
        self._routes_itself()
        ws = self._ws[n_tok]
        n, k, F, H = n_tok, self.k, self.F, self.H
        # the first 256 bytes hold the fused kernels' launch epoch, then the
        # per-expert-group kernel's row counters (8 tokens x H / 64 blocks)
        out, off = [], 256 + (4 * 8 * ((H + 63) // 64) + 255) // 256 * 256
        for count, dt, shape in ((n * k, torch.int32, (n, k)), (n * k, torch.float32, (n, k)),
                                 (n * k * F, torch.float32, (n, k, F)), (n * F, torch.float32, (n, F)),
                                 (n * k * H, torch.float32, (n, k, H)), (n * H, torch.float32, (n, H))):
            nbytes = 4 * count
            out.append(ws[off: off + nbytes].view(dt).view(shape))
            off += (nbytes + 255) // 256 * 256
        return tuple(out)

    def routing_of(self, n_tok):
        """(ids, weights) views of the last decode's routing in the workspace; with a
        router, the ids and weights of the last call (decode or prefill)."""
        if self.router is not None:
            return self._last(("routed", n_tok), n_tok)[3:]
        ids, w = self.intermediates(n_tok)[:2]
        return ids, w

    def _routes_itself(self):
        if self.router is not None:
            raise bad("a layer with a router keeps no such workspace: routing_of has the last call's ids and weights")

    def _last(self, key, n_tok):
        kept = self._ws.get(key)
        if kept is None:
            raise bad(f"the layer's last call was not one of {n_tok} tokens")
        return kept


class MXFP4Layer(MoELayer):
    """One MoE FFN layer whose experts are MXFP4 (gate, up and down alike), in
    device memory, laid out for the 4-bit tensor cores
    (moe_b200_mxfp4_layer_run). `router` (a Router) says how tokens pick their
    experts, None as MoELayer does: softmax, top-k. `biases` may hold f32
    "gate", "up" [E, F] and "down" [E, H]; `planes` MXFP4 planes hold every
    activation. `weights` as MoELayer's: ggml blocks, uint8 [E, rows, bytes] per
    role and [rows, bytes] for "shared_<role>" (whose F may be its own); None
    draws N(0, sigma)."""

    def __init__(self, H, F, n_experts, k, types, shared=True, glu_op=GLU_SWIGLU, glu_limit=0.0, norm_w=False, device="cuda",
                 host=False, name="blk.0", seed=0, weights=None, sigma=0.02, router=None, biases=None, planes=2):
        router = _checked_router(router, k, norm_w)
        self.types = dict(types)
        if set(self.types.values()) != {MXFP4}:
            raise bad("an MXFP4 layer has gate, up and down of type MXFP4")
        if host:
            raise bad("MXFP4 experts live in device memory")
        device = torch.device(device)
        if device.index is None:
            device = torch.device(device.type, torch.cuda.current_device())
        self.H, self.F, self.E, self.k, self.device, self.name = H, F, n_experts, k, device, name
        self.glu_op, self.glu_limit, self.norm_w, self.planes = glu_op, glu_limit, norm_w, planes
        self.router = Router(k, norm_w=norm_w) if router is None else router
        rb = self._router_bias = self.router.bias   # (kept: the descriptor points at it)
        if rb is not None and (rb.device != device or rb.shape[0] != n_experts):
            raise bad("the router's bias must be f32 [n_experts] on the layer's device")
        shapes = {"gate": (F, H), "up": (F, H), "down": (H, F)}
        gen = torch.Generator(device=device).manual_seed(seed)

        def blocks(key, n, rows, K):
            if weights is not None:
                b = torch.as_tensor(weights[key]).to(device)
                return b.reshape(n, *b.shape[-2:]).contiguous()
            return quantize_mxfp4(sigma * torch.randn((n, rows, K), generator=gen, device=device))
        self.w, self.shared, self.biases = {}, {}, {}
        for role, (rows, K) in shapes.items():
            self.w[role] = MXFP4Weights(blocks(role, n_experts, rows, K), K, rows)
        if shared and (weights is None or weights.get("shared_up") is not None):
            Fs = F if weights is None else torch.as_tensor(weights["shared_up"]).shape[-2]
            for role, (rows, K) in (("gate", (Fs, H)), ("up", (Fs, H)), ("down", (H, Fs))):
                self.shared[role] = MXFP4Weights(blocks(f"shared_{role}", 1, rows, K), K, rows)
        d = MoeMxfp4Layer()
        for role in shapes:
            setattr(d, role, self.w[role].desc)
            if self.shared:
                setattr(d, f"shared_{role}", self.shared[role].desc)
            b = (biases or {}).get(role)
            if b is not None:
                given(b, f"{role} bias", torch.float32, (n_experts, shapes[role][0]), device)
                self.biases[role] = b
                setattr(d, f"{role}_bias", b.data_ptr())
        d.k, d.glu_op, d.glu_limit, d.planes, d.router = k, glu_op, glu_limit, planes, self.router.desc
        d.router_bias = None if rb is None else rb.data_ptr()
        self.desc, self.ref = d, ctypes.byref(d)
        self._ws, self._ws_bytes = {}, {}       # the last call's workspace by its number of tokens; sizes

    def weight_bytes_per_token(self):
        """Expert bytes one batch-1 token streams: k routed + shared experts x 3 matrices."""
        per = sum(self.w[r].data.numel() // self.E for r in ("gate", "up", "down"))
        return per * self.k + sum(m.data.numel() for m in self.shared.values())

    def workspace(self, n_tok):
        """A call's workspace, from the current stream's memory (a capture's own within one): prompts come in
        any length, so the layer keeps the last call's only."""
        nbytes = self._ws_bytes.get(n_tok)
        if nbytes is None:
            if len(self._ws_bytes) >= 1024:
                self._ws_bytes.clear()
            nbytes = self._ws_bytes[n_tok] = lib().moe_b200_mxfp4_layer_workspace_size(self.ref, n_tok)
        self._ws = {}
        ws = self.w["up"].data.new_empty(nbytes)
        self._ws = {n_tok: ws}
        return ws

    def fused(self, n_tok):
        return False

    def decode(self, x, logits, out=None, stream=None, trace=None):
        """x f32 / f16 / bf16 [n_tok, H], logits f32 / f16 / bf16 [n_tok, E] -> out f32
        [n_tok, H], for one token or a prompt. Every call has a workspace of its own,
        so calls may overlap on the GPU. `trace` as MoELayer.decode."""
        xs, ls = dense_rows(x, "x"), dense_rows(logits, "logits")
        n_tok, dev = x.shape[0], self.device
        if tuple(x.shape) != (n_tok, self.H) or tuple(logits.shape) != (n_tok, self.E) or x.device != dev or logits.device != dev:
            raise bad("x must be [n_tok, H] and logits [n_tok, n_experts] on the layer's device")
        ctx, st = on(dev, stream)
        with ctx:
            out = x.new_empty((n_tok, self.H), dtype=torch.float32) if out is None else \
                given(out, "out", torch.float32, (n_tok, self.H), dev)
            if n_tok:
                ws = self.workspace(n_tok)
                check(lib().moe_b200_mxfp4_layer_run(self.ref, x.data_ptr(), ELEM[x.dtype], xs, logits.data_ptr(),
                                                     ELEM[logits.dtype], ls, out.data_ptr(), n_tok, ws.data_ptr(), ws.numel(), st))
            picks = self.routing_of(n_tok)[0].cpu().numpy() if trace is not None and n_tok else None
        if stream is not None:
            keep(stream, x, logits, out, self._router_bias, *self.biases.values(), *(m.data for m in self.w.values()),
                 *(m.data for m in self.shared.values()))
        if picks is not None:
            for r in ("gate", "up", "down"):
                trace.record(f"{self.name}.ffn_{r}_exps.weight", picks, self.E)
        return out

    prefill = decode

    def intermediates(self, n_tok):
        """Views of the last call's workspace: ids [n][k], weights [n][k], h [n][k][F]
        (GLU output), y [n][k][H] (down outputs)."""
        ws, n, k = self._last(n_tok, n_tok), n_tok, self.k
        out, off = [], 0
        for dt, shape in ((torch.int32, (n, k)), (torch.float32, (n, k)), (torch.float32, (n, k, self.F)),
                          (torch.float32, (n, k, self.H))):
            nbytes = 4 * math.prod(shape)
            out.append(ws[off: off + nbytes].view(dt).view(shape))
            off += (nbytes + 255) // 256 * 256
        return tuple(out)

    def routing_of(self, n_tok):
        """(ids, weights) views of the last call's routing in the workspace."""
        return self.intermediates(n_tok)[:2]


class Stack:
    """Batch-1 layers decoded back to back in one persistent launch
    (moe_b200_stack_prepare / moe_b200_stack_run). Layer l reads xs[l] and
    logits[l] (device f32 [1, H] / [1, E]), writes outs[l] and, with
    x_nexts, x_nexts[l] = xs[l] + outs[l] (a residual chain when xs[l + 1]
    is x_nexts[l]). The layers share one shape; their types are either one
    type for every tensor or, per layer, gate = up with the gate/up and down
    types among Q2_K, Q3_K, Q4_K, Q6_K (the mixed-type kernel); layers with a
    router of their own, MXFP4 ones among them, are refused. run() may be
    repeated; every tensor must stay alive."""

    def __init__(self, layers, xs, logits, outs, x_nexts=None, stream=None):
        n = len(layers)
        if any(getattr(L, "router", None) is not None for L in layers):
            raise bad("the stack kernel routes by softmax, top-k: it takes no layer with a router of its own")
        self.layers, self.n = layers, n
        self.desc0 = layers[0].desc
        arr = (MoeLayerDesc * n)(*[L.desc for L in layers])
        nbytes = lib().moe_b200_stack_workspace_size(ctypes.byref(self.desc0), n)
        self.ws = torch.zeros(nbytes, dtype=torch.uint8, device=layers[0].device)

        def ptrs(ts):
            return (ctypes.c_void_p * n)(*[_ptr(t) for t in ts])
        check(lib().moe_b200_stack_prepare(arr, n, ptrs(xs), ptrs(logits), ptrs(outs),
                                           ptrs(x_nexts) if x_nexts is not None else None, _ptr(self.ws),
                                           self.ws.numel(), _stream(stream)))

    def run(self, stream=None):
        check(lib().moe_b200_stack_run(ctypes.byref(self.desc0), self.n, _ptr(self.ws), self.ws.numel(),
                                       _stream(stream)))

