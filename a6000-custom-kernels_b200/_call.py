"""What the tensor-level calls share: the device and stream they run on, and
their checks of arguments. Kept short: for one token a call's host time is its
time."""
import contextlib

import torch
from torch.autograd import forward_ad

from ._lib import MOE_ERR_INVALID, MoeError
from .moe_cache import BF16, F16, F32

ELEM = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_HERE = contextlib.nullcontext()
_raw_stream = torch._C._cuda_getCurrentRawStream


def bad(msg):
    return MoeError(MOE_ERR_INVALID, msg)


def on(device, stream):
    """(context, raw handle) of a call on `device`: its current stream, or
    `stream` (a torch.cuda.Stream or a raw handle), which the context makes
    current so that what the call allocates belongs to it."""
    index = device.index
    if stream is None:
        if index == torch.cuda.current_device():
            return _HERE, _raw_stream(index)
        return torch.cuda.device(device), _raw_stream(index)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device)
    elif stream.device != device:
        raise bad(f"stream on {stream.device}, tensors on {device}")
    return torch.cuda.stream(stream), stream.cuda_stream


def keep(stream, *tensors):
    """The memory of what a call on `stream` (a torch.cuda.Stream that the caller
    named) uses is not handed out again before the stream has run the call.
    Nothing for a raw handle: its owner may destroy the stream first, so the
    caller keeps the tensors."""
    if stream is not None and not isinstance(stream, int):
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def no_tangents(*tensors):
    """Refuses tensors with a forward-mode derivative, which a call would drop. (They exist where
    forward_ad._current_level >= 0: calls look at that themselves.)"""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise bad("forward-mode derivatives are not offered")


def dense_rows(x, name):
    """Row stride in elements of a device tensor of F32, F16 or BF16 whose last
    dimension is dense and whose rows step evenly in memory."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise bad(f"{name} must be a CUDA tensor")
    if x.dtype not in ELEM:
        raise bad(f"{name} must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() < 2:
        raise bad(f"{name} needs at least two dimensions")
    K = x.shape[-1]
    if x.is_contiguous():
        return K
    if x.numel() == 0:
        return K
    if x.stride(-1) != 1 and K != 1:
        raise bad(f"{name}'s last dimension must be dense")
    stride, span = None, 1
    for size, st in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride = st
        if st != stride * span:
            raise bad(f"{name}'s rows must step evenly in memory")
        span *= size
    if stride is None:
        return K
    if stride < K:
        raise bad(f"{name}'s rows overlap in memory")
    return stride


def given(t, name, dtype, shape, device):
    """A contiguous tensor that the caller brought for an output."""
    if t.dtype != dtype or t.device != device or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise bad(f"{name} must be contiguous {dtype} {tuple(shape)} on {device}")
    return t
