"""4-bit matrices with a scale (and a zero) per group of values, and their products
with a few tokens (include/moe_cache_b200.h): value = scale * (code - zero).

Streams, outputs and workspaces as in mxfp4.py: `stream` is a torch.cuda.Stream, a
raw handle, or None for the device's current stream; what a call makes is allocated
there; with a raw handle the caller keeps the tensors until the stream has run it.

The products have no derivatives. Where gradients are recorded and x or a bias requires
one, a result says so (it requires grad, too), and a backward pass through it is refused;
with `dst` the call itself is. Forward-mode derivatives are refused.
"""
import ctypes

import torch
from torch.autograd import forward_ad

from ._call import ELEM, bad, dense_rows, given, keep, no_tangents, on
from ._lib import MoeW4, check, lib
from .moe_cache import BF16, F16, GLU_SWIGLU

_SCALES = {torch.float16: F16, torch.bfloat16: BF16}


class W4Weights:
    """A matrix, or the matrices of a layer's experts, laid out once for the product:
    `codes` uint8 [E, rows, ceil(K / 2)] or [rows, ceil(K / 2)] (value 2 i in the low
    nibble of byte i), `scales` f16 / bf16 [..., rows, ceil(K / group)], `zeros` uint8 of
    that shape (0 to 127; None: 8). `group` is a power of two from 32 on, or at least K
    (one group a row). The sources may be dropped afterwards; calls on other streams
    than `stream` wait for it as for any tensor made there.

    `data` is the laid-out bytes, for copies and broadcasts of them. Products read them ahead of
    the end of the kernel before them; so once `data` has been asked for, which may be to
    write it, products pay for a small launch that keeps them behind whatever did, until
    settle() is called behind the last write."""

    def __init__(self, codes, scales, K, group, zeros=None, stream=None):
        for t, name, types in ((codes, "codes", (torch.uint8,)), (scales, "scales", tuple(_SCALES)), (zeros, "zeros", (torch.uint8,))):
            if t is None and name == "zeros":
                continue
            if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in types and t.is_contiguous() and t.dim() in (2, 3)):
                raise bad(f"{name} must be a contiguous {' / '.join(str(d)[6:] for d in types)} CUDA tensor [E, rows, n] or [rows, n]")
            if t.device != codes.device or t.shape[:-1] != codes.shape[:-1]:
                raise bad(f"{name} must have the codes' device, experts and rows")
        if K < 1 or group < 1 or codes.shape[-1] != (K + 1) // 2:
            raise bad("codes must hold ceil(K / 2) bytes a row, K >= 1 and group >= 1")
        n = -(-K // group)
        if scales.shape[-1] != n or (zeros is not None and zeros.shape[-1] != n):
            raise bad("scales and zeros must hold ceil(K / group) groups a row")
        self.E, self.rows = codes.shape[0] if codes.dim() == 3 else 1, codes.shape[-2]
        self.K, self.group, self.device = K, group, codes.device
        self.desc = MoeW4(None, self.E, self.rows, K, group, _SCALES[scales.dtype], zeros is not None)
        self.ref = ctypes.byref(self.desc)
        ctx, st = on(self.device, stream)
        with ctx:
            self._data = codes.new_empty(max(1, lib().moe_b200_w4_packed_size(self.ref)))
            check(lib().moe_b200_w4_pack(self.ref, codes.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
                                         self._data.data_ptr(), self._data.numel(), st))
        self.desc.data = self._data.data_ptr()
        self._open = False       # whether others may have written _data
        keep(stream, codes, scales, zeros)
        self.shape = (self.E, self.rows, K, group, scales.dtype, zeros is not None, self.device)
        self._ws_bytes = {}      # workspace sizes by call

    @property
    def data(self):
        self._open = True
        return self._data

    def settle(self, stream=None):
        """Behind the last write to `data`, on its stream: products need no launch of their own for it any longer."""
        ctx, st = on(self.device, stream)
        with ctx:
            check(lib().moe_b200_w4_settle(st))
        self._open = False


def w4_workspace_size(w, n_tok, k, dtype, per_pick=False):
    """Bytes of device workspace that w4_mul_mat (k = 0) or w4_mul_mat_id need (moe_b200_w4_workspace_size): 0 for few
    rows of x. per_pick: x is [n_tok, k, K]."""
    n = w._ws_bytes.get((n_tok, k, dtype, per_pick))
    if n is None:
        if len(w._ws_bytes) >= 1024:
            w._ws_bytes.clear()
        n = w._ws_bytes[n_tok, k, dtype, per_pick] = lib().moe_b200_w4_workspace_size(w.ref, n_tok, k, ELEM[dtype], per_pick)
    return n


def _workspace(workspace, w, x, *call):
    """(tensor, address, bytes) of a call's workspace: the caller's, or one of its own where it needs one."""
    if workspace is None:
        n = w4_workspace_size(w, *call)
        if n == 0:
            return None, None, 0
        workspace = x.new_empty(n, dtype=torch.uint8)
        return workspace, workspace.data_ptr(), n
    if not isinstance(workspace, torch.Tensor) or workspace.dtype != torch.uint8 or workspace.device != w.device or \
            not workspace.is_contiguous():
        raise bad("workspace must be contiguous uint8 on the weights' device")
    return workspace, workspace.data_ptr(), workspace.numel()


def _bias(b, name, w):
    if b is None:
        return None
    if not isinstance(b, torch.Tensor) or b.dtype != torch.float32 or b.device != w.device or not b.is_contiguous() or \
            (tuple(b.shape) != (w.E, w.rows) and (w.E != 1 or tuple(b.shape) != (w.rows,))):
        raise bad(f"{name} must be contiguous f32 [n_experts, rows] on the weights' device")
    return b.data_ptr()


def _gate(gate, gate_bias, w):
    if gate is not None:
        if gate.shape != w.shape:
            raise bad("gate must have w's shape, group, scale type, zeros and device")
    elif gate_bias is not None:
        raise bad("gate_bias without a gate")


class _NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, args, *inputs):
        return call(*args)

    @staticmethod
    def backward(ctx, g):
        raise bad("products with 4-bit matrices have no gradient: detach their inputs, or call them under torch.no_grad()")


def _wants_grad(dst, *inputs):
    """Whether a call's result has to carry that it depends on these inputs."""
    if forward_ad._current_level >= 0:
        no_tangents(*inputs)
    if not (any(t is not None and t.requires_grad for t in inputs) and torch.is_grad_enabled()):
        return False
    if dst is not None:
        raise bad("with dst an input that requires a gradient is refused: detach it, or call under torch.no_grad()")
    return True


def w4_mul_mat(w, x, gate=None, bias=None, gate_bias=None, glu_op=GLU_SWIGLU, glu_limit=0.0, dst=None, workspace=None,
               stream=None):
    """x f32 / f16 / bf16 [n_tok, K] times one 4-bit matrix (W4Weights with E = 1) -> dst f32
    [n_tok, rows] = w . x (+ bias), or GLU(gate . x + gate_bias, w . x + bias) with
    `gate`. x is not quantised: f16 is exact, f32 is held to 2^-22 of a value, and f32 and
    bf16 to 2^-39 of the largest of 256. Sums are in 32 bits, of up to 128 values in the
    tensor cores; their errors are relative to the sum of |scale| (code + zero) |x|. Against
    64 bits a product with N(0, 1) x is off by 1e-7 to 4e-7 (2-norm); a row's last bits may
    change with n_tok. A NaN or an infinity in a row of x makes that row's outputs NaN."""
    stride = dense_rows(x, "x")
    dev, n_tok = w.device, x.shape[0]
    if w.E != 1:
        raise bad("w holds several matrices: w4_mul_mat_id takes the experts' ids")
    if x.dim() != 2 or x.shape[1] != w.K or x.device != dev:
        raise bad(f"x must be [n_tok, {w.K}] on the weights' device")
    _gate(gate, gate_bias, w)
    b, gb = _bias(bias, "bias", w), _bias(gate_bias, "gate_bias", w)
    # (what _wants_grad asks is true of few calls)
    if (x.requires_grad or forward_ad._current_level >= 0 or (bias is not None and bias.requires_grad) or
            (gate_bias is not None and gate_bias.requires_grad)) and _wants_grad(dst, x, bias, gate_bias):
        # (no closure: its variables would cost every call 0.3 us)
        return _NoGradient.apply(w4_mul_mat, (w, x, gate, bias, gate_bias, glu_op, glu_limit, None, workspace, stream),
                                 x, bias, gate_bias)
    ctx, st = on(dev, stream)
    with ctx:
        dst = x.new_empty((n_tok, w.rows), dtype=torch.float32) if dst is None else \
            given(dst, "dst", torch.float32, (n_tok, w.rows), dev)
        workspace, ws_ptr, ws_bytes = _workspace(workspace, w, x, n_tok, 0, x.dtype)
        if w._open or (gate is not None and gate._open):
            check(lib().moe_b200_w4_settle(st))
        check(lib().moe_b200_w4_mul_mat_id(w.ref, None if gate is None else gate.ref, b, gb, glu_op, glu_limit, x.data_ptr(),
                                           ELEM[x.dtype], stride, 0, n_tok, None, 1, 1, dst.data_ptr(), ws_ptr, ws_bytes, st))
    if stream is not None:
        keep(stream, w._data, None if gate is None else gate._data, x, bias, gate_bias, dst, workspace)
    return dst


def w4_mul_mat_id(w, x, ids, gate=None, bias=None, gate_bias=None, glu_op=GLU_SWIGLU, glu_limit=0.0, dst=None, workspace=None,
                  stream=None):
    """MUL_MAT_ID of 4-bit experts (moe_b200_w4_mul_mat_id): x f32 / f16 / bf16 [n_tok, K],
    or [n_tok, k, K] with a row per pick, ids i32 [n_tok, k] -> dst f32 [n_tok, k, rows] =
    experts w . x (+ bias), or GLU(gate . x + gate_bias, w . x + bias) with `gate`. Picks
    with id -1 leave their rows of dst as they were. x and sums are held as in w4_mul_mat."""
    if not (isinstance(ids, torch.Tensor) and ids.is_cuda and ids.dtype == torch.int32 and ids.dim() == 2):
        raise bad("ids must be an i32 CUDA tensor [n_tok, k]")
    n_tok, k = ids.shape
    ids_stride = k
    if not ids.is_contiguous() and n_tok > 0:
        ids_stride = ids.stride(0) if n_tok > 1 else k
        if (ids.stride(1) != 1 and k > 1) or ids_stride < k:
            raise bad("ids' rows must be dense and must not overlap in memory")
    stride = dense_rows(x, "x")
    per_pick = x.dim() == 3
    dev, K, rows = w.device, w.K, w.rows
    if tuple(x.shape) != ((n_tok, k, K) if per_pick else (n_tok, K)):
        raise bad(f"x must be [n_tok, {K}] or [n_tok, k, {K}]")
    if x.device != dev or ids.device != dev:
        raise bad("x, ids and the weights must be on one device")
    _gate(gate, gate_bias, w)
    b, gb = _bias(bias, "bias", w), _bias(gate_bias, "gate_bias", w)
    # (what _wants_grad asks is true of few calls)
    if (x.requires_grad or forward_ad._current_level >= 0 or (bias is not None and bias.requires_grad) or
            (gate_bias is not None and gate_bias.requires_grad)) and _wants_grad(dst, x, bias, gate_bias):
        return _NoGradient.apply(w4_mul_mat_id, (w, x, ids, gate, bias, gate_bias, glu_op, glu_limit, None, workspace, stream),
                                 x, bias, gate_bias)
    ctx, st = on(dev, stream)
    with ctx:
        dst = x.new_empty((n_tok, k, rows), dtype=torch.float32) if dst is None else \
            given(dst, "dst", torch.float32, (n_tok, k, rows), dev)
        workspace, ws_ptr, ws_bytes = _workspace(workspace, w, x, n_tok, k, x.dtype, per_pick)
        if w._open or (gate is not None and gate._open):
            check(lib().moe_b200_w4_settle(st))
        check(lib().moe_b200_w4_mul_mat_id(w.ref, None if gate is None else gate.ref, b, gb, glu_op, glu_limit, x.data_ptr(),
                                           ELEM[x.dtype], stride, per_pick, n_tok, ids.data_ptr(), k, ids_stride,
                                           dst.data_ptr(), ws_ptr, ws_bytes, st))
    if stream is not None:
        keep(stream, w._data, None if gate is None else gate._data, x, ids, bias, gate_bias, dst, workspace)
    return dst


__all__ = ["W4Weights", "w4_mul_mat", "w4_mul_mat_id", "w4_workspace_size"]
