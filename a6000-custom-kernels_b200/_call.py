"""What the tensor-level calls share: the device and stream they run on, and
their checks of arguments."""
import torch

from ._lib import MOE_ERR_INVALID, MoeError
from .moe_cache import BF16, F16, F32

ELEM = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class On:
    """The call's device and stream: enters both, and gives the stream's handle."""

    def __init__(self, device, stream):
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=device)
        elif stream is not None and stream.device != device:
            raise MoeError(MOE_ERR_INVALID, f"stream on {stream.device}, tensors on {device}")
        self.device, self.stream = device, stream
        self.ctx = None

    def __enter__(self):
        current = torch.cuda.current_stream(self.device)
        if self.stream is not None and self.stream != current:
            self.ctx = torch.cuda.stream(self.stream)      # sets the device too
        elif self.device.index != torch.cuda.current_device():
            self.ctx = torch.cuda.device(self.device)
        if self.ctx is not None:
            self.ctx.__enter__()
        return (self.stream or current).cuda_stream

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)


def need(cond, msg):
    if not cond:
        raise MoeError(MOE_ERR_INVALID, msg)


def dense_rows(x, name, dtypes):
    """A device tensor whose last dimension is dense and whose leading ones step evenly: (row stride, rows)."""
    need(isinstance(x, torch.Tensor) and x.is_cuda, f"{name} must be a CUDA tensor")
    need(x.dtype in dtypes, f"{name} must be one of {[str(d) for d in dtypes]}, got {x.dtype}")
    need(x.dim() >= 2, f"{name} needs at least two dimensions")
    K = x.shape[-1]
    n = x.numel() // K if K else 0
    if n <= 1:
        need(n == 0 or x.stride(-1) == 1 or K == 1, f"{name}'s last dimension must be dense")
        return K, n
    need(x.stride(-1) == 1 or K == 1, f"{name}'s last dimension must be dense")
    stride, span = None, 1
    for size, st in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride = st
        need(st == stride * span, f"{name}'s rows must step evenly in memory")
        span *= size
    need(stride >= K, f"{name}'s rows overlap in memory")
    return stride, n
