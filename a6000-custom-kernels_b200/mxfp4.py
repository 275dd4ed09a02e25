"""MXFP4 experts: the quantiser and its read-back, expert matrices laid out for
the 4-bit tensor cores, and their MUL_MAT_ID (include/moe_cache_b200.h).

Every call checks its tensors (device, type, contiguity) and works on the
tensors' device; `stream` is a torch.cuda.Stream, a raw handle, or None for the
device's current stream. Outputs and workspaces that a call makes are taken
from the allocator for that stream.
"""
import ctypes

import torch

from ._call import ELEM, On, dense_rows, need
from ._lib import MoeMxfp4, MoeTensor, check, lib
from .moe_cache import GLU_SWIGLU, MXFP4, TSIZE, row_size


def quantize_mxfp4(x, planes=1, out=None, stream=None):
    """f32 / f16 / bf16 [..., K] -> uint8 MXFP4 blocks [..., 17 K / 32], or
    [planes, ..., 17 K / 32] with planes = 2 (plane 1: what plane 0 leaves of
    x). K a multiple of 32; rows may lie in a wider buffer."""
    stride, n = dense_rows(x, "x", ELEM)
    K = x.shape[-1]
    need(K > 0 and K % 32 == 0, "K must be a positive multiple of 32")
    need(planes in (1, 2), "planes must be 1 or 2")
    shape = ((planes,) if planes > 1 else ()) + tuple(x.shape[:-1]) + (row_size(MXFP4, K),)
    with On(x.device, stream) as st:
        if out is None:
            out = torch.empty(shape, dtype=torch.uint8, device=x.device)
        else:
            need(out.dtype == torch.uint8 and out.device == x.device and tuple(out.shape) == shape and
                  out.is_contiguous(), f"out must be contiguous uint8 {shape} on {x.device}")
        check(lib().moe_b200_quantize_mxfp4(x.data_ptr(), ELEM[x.dtype], n, K, max(stride, K), planes, out.data_ptr(), st))
    return out


def dequantize_mxfp4(blocks, K, planes=None, dtype=torch.float32, out=None, stream=None):
    """The values of quantize_mxfp4's blocks: [..., K] in `dtype`. `planes` says
    whether the first dimension counts planes; None takes it for the planes
    when `blocks` has three dimensions and the first is 2."""
    need(isinstance(blocks, torch.Tensor) and blocks.is_cuda and blocks.dtype == torch.uint8 and
          blocks.is_contiguous() and blocks.dim() >= 2, "blocks must be a contiguous uint8 CUDA tensor of two or more dimensions")
    need(K > 0 and K % 32 == 0 and blocks.shape[-1] == row_size(MXFP4, K), "blocks' last dimension must hold K values")
    if planes is None:
        planes = 2 if blocks.dim() == 3 and blocks.shape[0] == 2 else 1
    need(planes == 1 or (planes == 2 and blocks.dim() >= 3 and blocks.shape[0] == 2), "planes must be 1, or 2 with blocks [2, ..., bytes]")
    need(dtype in ELEM, "dtype must be float32, float16 or bfloat16")
    shape = tuple(blocks.shape[1 if planes == 2 else 0:-1]) + (K,)
    with On(blocks.device, stream) as st:
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=blocks.device)
        else:
            need(out.dtype == dtype and tuple(out.shape) == shape and out.device == blocks.device,
                  f"out must be {dtype} {shape} on {blocks.device}")
        stride, n = dense_rows(out, "out", ELEM)
        check(lib().moe_b200_dequantize_mxfp4(blocks.data_ptr(), n, K, planes, out.data_ptr(), ELEM[dtype], max(stride, K), st))
    return out


class MXFP4Weights:
    """The matrices of a layer's experts, laid out once for the 4-bit tensor
    cores from ggml MXFP4 blocks (uint8 [E, rows, 17 K / 32], on the device).
    `blocks` may be dropped afterwards."""

    def __init__(self, blocks, K, rows, stream=None):
        need(isinstance(blocks, torch.Tensor) and blocks.is_cuda and blocks.dtype == torch.uint8 and
              blocks.is_contiguous() and blocks.dim() == 3, "blocks must be a contiguous uint8 CUDA tensor [E, rows, 17 K / 32]")
        need(K > 0 and K % 32 == 0 and tuple(blocks.shape[1:]) == (rows, row_size(MXFP4, K)),
              "blocks must be [E, rows, 17 K / 32]")
        self.E, self.rows, self.K, self.device = blocks.shape[0], rows, K, blocks.device
        t = MoeTensor()
        t.data, t.type = blocks.data_ptr(), MXFP4
        rb = row_size(MXFP4, K)
        t.ne[0], t.ne[1], t.ne[2], t.ne[3] = K, rows, self.E, 1
        t.nb[0], t.nb[1], t.nb[2], t.nb[3] = TSIZE[MXFP4], rb, rb * rows, rb * rows * self.E
        with On(self.device, stream) as st:
            self.data = torch.empty(max(1, lib().moe_b200_mxfp4_packed_size(self.E, rows, K)), dtype=torch.uint8,
                                    device=self.device)
            check(lib().moe_b200_mxfp4_pack(ctypes.byref(t), self.data.data_ptr(), self.data.numel(), st))
        self.desc = MoeMxfp4(self.data.data_ptr(), self.E, rows, K)
        self.ref = ctypes.byref(self.desc)


def mxfp4_workspace_size(w, n_tok, k, planes=2):
    """Bytes of device workspace mxfp4_mul_mat_id needs (moe_b200_mxfp4_workspace_size)."""
    return lib().moe_b200_mxfp4_workspace_size(w.ref, n_tok, k, planes)


def mxfp4_mul_mat_id(w, x, ids, gate=None, bias=None, gate_bias=None, glu_op=GLU_SWIGLU, glu_limit=0.0, planes=2,
                     dst=None, workspace=None, stream=None):
    """MUL_MAT_ID of MXFP4 experts (moe_b200_mxfp4_mul_mat_id): x f32 / f16 / bf16
    [n_tok, K], or [n_tok, k, K] with a row per pick, ids i32 [n_tok, k] -> dst
    f32 [n_tok, k, rows] = experts w . x (+ bias), or GLU(gate . x + gate_bias,
    w . x + bias) with `gate`. Picks with id -1 leave their rows of dst as they
    were; `planes` MXFP4 planes hold x (2: about three decimal digits)."""
    need(isinstance(ids, torch.Tensor) and ids.is_cuda and ids.dtype == torch.int32 and ids.dim() == 2 and
          (ids.stride(1) == 1 or ids.shape[1] == 1), "ids must be an i32 CUDA tensor [n_tok, k] with dense rows")
    n_tok, k = ids.shape
    need(k >= 1, "ids needs at least one pick per token")
    need(n_tok <= 1 or ids.stride(0) >= k, "ids' rows overlap in memory")
    per_pick = isinstance(x, torch.Tensor) and x.dim() == 3
    stride, _ = dense_rows(x, "x", ELEM)
    K, rows = w.K, w.rows
    need(tuple(x.shape) == ((n_tok, k, K) if per_pick else (n_tok, K)), f"x must be [n_tok, {K}] or [n_tok, k, {K}]")
    need(x.device == w.device and ids.device == w.device, "x, ids and the weights must be on one device")
    if gate is not None:
        need((gate.E, gate.rows, gate.K, gate.device) == (w.E, rows, K, w.device), "gate must have w's shape and device")
    else:
        need(gate_bias is None, "gate_bias without a gate")
    for name, b in (("bias", bias), ("gate_bias", gate_bias)):
        need(b is None or (b.dtype == torch.float32 and b.device == w.device and b.is_contiguous() and
                            tuple(b.shape) == (w.E, rows)), f"{name} must be contiguous f32 [n_experts, rows]")
    with On(w.device, stream) as st:
        L = lib()
        if dst is None:
            dst = torch.empty((n_tok, k, rows), dtype=torch.float32, device=w.device)
        else:
            need(dst.dtype == torch.float32 and dst.device == w.device and dst.is_contiguous() and
                  tuple(dst.shape) == (n_tok, k, rows), "dst must be contiguous f32 [n_tok, k, rows]")
        if workspace is None:
            workspace = torch.empty(L.moe_b200_mxfp4_workspace_size(w.ref, n_tok, k, planes) or 1,
                                    dtype=torch.uint8, device=w.device)
        else:
            need(workspace.dtype == torch.uint8 and workspace.device == w.device and workspace.is_contiguous(),
                  "workspace must be contiguous uint8 on the weights' device")
        check(L.moe_b200_mxfp4_mul_mat_id(
            w.ref, gate.ref if gate is not None else None, None if bias is None else bias.data_ptr(),
            None if gate_bias is None else gate_bias.data_ptr(), glu_op, glu_limit, x.data_ptr(), ELEM[x.dtype],
            max(stride, K), int(per_pick), n_tok, ids.data_ptr(), k, max(ids.stride(0), k), planes, dst.data_ptr(),
            workspace.data_ptr(), workspace.numel(), st))
    return dst


__all__ = ["quantize_mxfp4", "dequantize_mxfp4", "MXFP4Weights", "mxfp4_mul_mat_id", "mxfp4_workspace_size"]