"""MXFP4 experts: the quantiser and its read-back, expert matrices laid out for
the 4-bit tensor cores, and their MUL_MAT_ID (include/moe_cache_b200.h).

Every call checks its tensors (device, type, layout; MoeError otherwise) and
works on the tensors' device; `stream` is a torch.cuda.Stream, a raw handle, or
None for the device's current stream. Outputs and workspaces that a call makes
are allocated on that stream. Inputs must be ready there; with a
torch.cuda.Stream they may be dropped right behind the call, with a raw handle
the caller keeps them until the stream has run it.
"""
import ctypes

import torch

from ._call import ELEM, bad, dense_rows, given, keep, on
from ._lib import MoeMxfp4, MoeTensor, check, lib
from .moe_cache import GLU_SWIGLU, MXFP4, TSIZE, row_size


def _version(t):
    """What changes when something else writes t (inference tensors do not count)."""
    return None if t.is_inference() else t._version


def quantize_mxfp4(x, planes=1, out=None, stream=None):
    """f32 / f16 / bf16 [..., K] -> uint8 MXFP4 blocks [..., 17 K / 32], or
    [planes, ..., 17 K / 32] with planes = 2 (plane 1: what plane 0 leaves of
    x). K a multiple of 32; rows may lie in a wider buffer."""
    stride = dense_rows(x, "x")
    K = x.shape[-1]
    if K == 0 or K % 32:
        raise bad("K must be a positive multiple of 32")
    if planes not in (1, 2):
        raise bad("planes must be 1 or 2")
    shape = (*x.shape[:-1], K // 32 * 17)
    if planes == 2:
        shape = (2, *shape)
    ctx, st = on(x.device, stream)
    with ctx:
        if out is None:
            out, known = x.new_empty(shape, dtype=torch.uint8), True
        else:
            known = not given(out, "out", torch.uint8, shape, x.device).is_inference()
            if known:                          # other views of it see that it is written
                torch.autograd.graph.increment_version(out)
        check(lib().moe_b200_quantize_mxfp4(x.data_ptr(), ELEM[x.dtype], x.numel() // K, K, stride, planes, out.data_ptr(), st))
    keep(stream, x, out)
    if len(shape) > 2 and shape[0] == 2:      # two planes or two matrices: only this call knows
        out._mxfp4_planes = (planes, _version(out)) if known else (None, None)
    return out


def dequantize_mxfp4(blocks, K, planes=None, dtype=torch.float32, out=None, stream=None):
    """The values of quantize_mxfp4's blocks: [..., K] in `dtype`. `planes` = 2 says
    that the first dimension counts planes. None reads a tensor as the call of
    quantize_mxfp4 that returned it made it, and anything else as one plane --
    unless it has a first dimension of 2 before the rows, which could be either:
    that is refused."""
    if not (isinstance(blocks, torch.Tensor) and blocks.is_cuda and blocks.dtype == torch.uint8 and
            blocks.is_contiguous() and blocks.dim() >= 2):
        raise bad("blocks must be a contiguous uint8 CUDA tensor of two or more dimensions")
    shape = blocks.shape
    if K <= 0 or K % 32 or shape[-1] != K // 32 * 17:
        raise bad("blocks' last dimension must hold K values, K a multiple of 32")
    if planes is None:
        planes = 1
        if len(shape) > 2 and shape[0] == 2:
            planes, version = getattr(blocks, "_mxfp4_planes", (None, None))
            if planes is None or version != _version(blocks):
                raise bad("blocks with a first dimension of 2 may be two planes or two matrices: say planes=1 or planes=2")
    if planes != 1 and not (planes == 2 and len(shape) >= 3 and shape[0] == 2):
        raise bad("planes must be 1, or 2 with blocks [2, ..., bytes]")
    if dtype not in ELEM:
        raise bad("dtype must be float32, float16 or bfloat16")
    shape = (*shape[planes - 1:-1], K)
    ctx, st = on(blocks.device, stream)
    with ctx:
        if out is None:
            out, stride = blocks.new_empty(shape, dtype=dtype), K
        else:
            stride = dense_rows(out, "out")
            if out.dtype != dtype or tuple(out.shape) != shape or out.device != blocks.device:
                raise bad(f"out must be {dtype} {shape} on {blocks.device}")
        check(lib().moe_b200_dequantize_mxfp4(blocks.data_ptr(), out.numel() // K, K, planes, out.data_ptr(), ELEM[dtype],
                                              stride, st))
    keep(stream, blocks, out)
    return out


class MXFP4Weights:
    """The matrices of a layer's experts, laid out once for the 4-bit tensor
    cores from ggml MXFP4 blocks (uint8 [E, rows, 17 K / 32], on the device).
    `blocks` may be dropped afterwards (as the inputs of every call here); calls on
    other streams than `stream` wait for it as for any tensor made there."""

    def __init__(self, blocks, K, rows, stream=None):
        if not (isinstance(blocks, torch.Tensor) and blocks.is_cuda and blocks.dtype == torch.uint8 and
                blocks.is_contiguous() and blocks.dim() == 3):
            raise bad("blocks must be a contiguous uint8 CUDA tensor [E, rows, 17 K / 32]")
        if K <= 0 or K % 32 or tuple(blocks.shape[1:]) != (rows, row_size(MXFP4, K)):
            raise bad("blocks must be [E, rows, 17 K / 32], K a multiple of 32")
        self.E, self.rows, self.K, self.device = blocks.shape[0], rows, K, blocks.device
        t = MoeTensor()
        t.data, t.type = blocks.data_ptr(), MXFP4
        rb = row_size(MXFP4, K)
        t.ne[0], t.ne[1], t.ne[2], t.ne[3] = K, rows, self.E, 1
        t.nb[0], t.nb[1], t.nb[2], t.nb[3] = TSIZE[MXFP4], rb, rb * rows, rb * rows * self.E
        ctx, st = on(self.device, stream)
        with ctx:
            self.data = blocks.new_empty(max(1, lib().moe_b200_mxfp4_packed_size(self.E, rows, K)))
            check(lib().moe_b200_mxfp4_pack(ctypes.byref(t), self.data.data_ptr(), self.data.numel(), st))
        keep(stream, blocks)
        self.shape = (self.E, rows, K, self.device)
        self.desc = MoeMxfp4(self.data.data_ptr(), self.E, rows, K)
        self.ref = ctypes.byref(self.desc)
        self._ws_bytes = {}      # workspace sizes by (n_tok, k, planes)


def _workspace_bytes(w, *call):
    n = w._ws_bytes.get(call)
    if n is None:
        if len(w._ws_bytes) >= 1024:
            w._ws_bytes.clear()
        n = w._ws_bytes[call] = lib().moe_b200_mxfp4_workspace_size(w.ref, *call)
    return n


def mxfp4_workspace_size(w, n_tok, k, planes=2):
    """Bytes of device workspace mxfp4_mul_mat_id needs (moe_b200_mxfp4_workspace_size): 0 for a few tokens."""
    return _workspace_bytes(w, n_tok, k, planes)


def _bias(b, name, w):
    if b is None:
        return None
    if b.dtype != torch.float32 or b.device != w.device or not b.is_contiguous() or tuple(b.shape) != (w.E, w.rows):
        raise bad(f"{name} must be contiguous f32 [n_experts, rows] on the weights' device")
    return b.data_ptr()


def mxfp4_mul_mat_id(w, x, ids, gate=None, bias=None, gate_bias=None, glu_op=GLU_SWIGLU, glu_limit=0.0, planes=2,
                     dst=None, workspace=None, stream=None):
    """MUL_MAT_ID of MXFP4 experts (moe_b200_mxfp4_mul_mat_id): x f32 / f16 / bf16
    [n_tok, K], or [n_tok, k, K] with a row per pick, ids i32 [n_tok, k] -> dst
    f32 [n_tok, k, rows] = experts w . x (+ bias), or GLU(gate . x + gate_bias,
    w . x + bias) with `gate`. Picks with id -1 leave their rows of dst as they
    were; `planes` MXFP4 planes hold x."""
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
    if gate is not None:
        if gate.shape != w.shape:
            raise bad("gate must have w's shape and device")
    elif gate_bias is not None:
        raise bad("gate_bias without a gate")
    L = lib()
    ctx, st = on(dev, stream)
    with ctx:
        dst = x.new_empty((n_tok, k, rows), dtype=torch.float32) if dst is None else \
            given(dst, "dst", torch.float32, (n_tok, k, rows), dev)
        ws_ptr, ws_bytes = None, 0
        if workspace is None:
            ws_bytes = _workspace_bytes(w, n_tok, k, planes)
            if ws_bytes:
                workspace = x.new_empty(ws_bytes, dtype=torch.uint8)
                ws_ptr = workspace.data_ptr()
        elif workspace.dtype != torch.uint8 or workspace.device != dev or not workspace.is_contiguous():
            raise bad("workspace must be contiguous uint8 on the weights' device")
        else:
            ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel()
        check(L.moe_b200_mxfp4_mul_mat_id(
            w.ref, None if gate is None else gate.ref, _bias(bias, "bias", w), _bias(gate_bias, "gate_bias", w),
            glu_op, glu_limit, x.data_ptr(), ELEM[x.dtype], stride, per_pick, n_tok, ids.data_ptr(), k, ids_stride, planes,
            dst.data_ptr(), ws_ptr, ws_bytes, st))
    if stream is not None:
        keep(stream, w.data, None if gate is None else gate.data, x, ids, bias, gate_bias, dst, workspace)
    return dst


__all__ = ["quantize_mxfp4", "dequantize_mxfp4", "MXFP4Weights", "mxfp4_mul_mat_id", "mxfp4_workspace_size"]
