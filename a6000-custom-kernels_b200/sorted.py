"""Tokens sorted by expert and back (include/moe_cache_b200.h): the order of the
picks by expert, the tokens' rows in that order, and the weighted sum of such rows
back into the tokens, with gradients -- for experts that run outside this library.

    rows, order = dispatch_sorted(x, ids, n_experts)     # rows of expert e: order.offsets[e] to [e + 1]
    out = combine_sorted(experts(rows, order.offsets), order, weights)

`stream` is a torch.cuda.Stream, a raw handle, or None for the device's current
stream; outputs are allocated on it. With a torch.cuda.Stream the inputs may be
dropped right behind the call, with a raw handle the caller keeps them until the
stream has run it. gather_sorted, dispatch_sorted and combine_sorted are
differentiable once (in x, y, weights and shared); their backward pass runs on the
stream of the call.
"""
import torch
from torch.autograd.function import once_differentiable

from ._call import ELEM, bad, dense_rows, keep, on
from ._lib import check, lib


class ExpertOrder:
    """The picks of n_tok tokens by expert: `rows` i32 [n_tok k], the entry t k + j of
    each sorted row, and `experts`, its expert (-1 behind the last row); `positions`
    i32 [n_tok, k], the sorted row of a pick or -1; `offsets` i32 [n_experts + 1], the
    first sorted row of each expert, then their number."""

    def __init__(self, ids, n_experts, stream=None):
        if not (isinstance(ids, torch.Tensor) and ids.is_cuda and ids.dtype == torch.int32 and ids.dim() == 2):
            raise bad("ids must be an i32 CUDA tensor [n_tok, k]")
        n_tok, k = ids.shape
        stride = k
        if not ids.is_contiguous() and n_tok > 0:
            stride = ids.stride(0) if n_tok > 1 else k
            if (ids.stride(1) != 1 and k > 1) or stride < k:
                raise bad("ids' rows must be dense and must not overlap in memory")
        if k < 1 or n_experts < 1:
            raise bad("need k >= 1 and n_experts >= 1")
        ctx, st = on(ids.device, stream)
        n = n_tok * k
        with ctx:
            buf = ids.new_empty(3 * n + n_experts + 1)
            self.rows, pos, self.experts, self.offsets = buf.split([n, n, n, n_experts + 1])
            at = buf.data_ptr()
            check(lib().moe_b200_sort_by_expert(ids.data_ptr(), stride, n_tok, k, n_experts, at, at + 4 * n, at + 8 * n,
                                                at + 12 * n, st))
        self.positions = pos.view(n_tok, k)
        self.n_tok, self.k, self.n_experts, self.device = n_tok, k, n_experts, ids.device
        keep(stream, ids, buf)


def sort_by_expert(ids, n_experts, stream=None):
    """ids i32 [n_tok, k] (a Router's; -1: an empty slot) -> the ExpertOrder of its
    picks: by expert, and within one in the order of (token, pick)."""
    return ExpertOrder(ids, n_experts, stream)


def _tensors(order):
    """The order's tensors that the row calls read: positions, and the number of sorted rows behind the offsets."""
    return order.positions, order.offsets


def _gather(x, stride, positions, offsets, stream):
    n_tok, k = positions.shape
    H = x.shape[1]
    ctx, st = on(x.device, stream)
    with ctx:
        out = x.new_empty((n_tok * k, H))
        check(lib().moe_b200_gather_sorted(x.data_ptr(), ELEM[x.dtype], stride, n_tok, k, H, positions.data_ptr(),
                                           offsets.data_ptr() + 4 * (offsets.shape[0] - 1), out.data_ptr(), st))
    keep(stream, x, positions, offsets, out)
    return out


def _combine(y, stride, positions, weights, shared, shared_stride, stream):
    n_tok, k = positions.shape
    H = y.shape[1]
    ctx, st = on(y.device, stream)
    with ctx:
        out = y.new_empty((n_tok, H))
        check(lib().moe_b200_combine_sorted(y.data_ptr(), ELEM[y.dtype], stride, n_tok, k, H, positions.data_ptr(),
                                            None if weights is None else weights.data_ptr(),
                                            None if shared is None else shared.data_ptr(), shared_stride, out.data_ptr(), st))
    keep(stream, y, positions, weights, shared, out)
    return out


def _grad_rows(g):
    """A gradient as rows that the calls take (autograd may hand over an expanded one) and their stride."""
    if g.stride(1) != 1 or g.stride(0) < g.shape[1]:
        g = g.contiguous()
    return g, max(g.stride(0), g.shape[1])


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, stride, positions, offsets, stream):
        ctx.save_for_backward(positions)
        return _gather(x, stride, positions, offsets, stream)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        g, stride = _grad_rows(g)
        return _combine(g, stride, ctx.saved_tensors[0], None, None, 0, None), None, None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, stride, positions, offsets, weights, shared, shared_stride, stream):
        need_y = y if weights.requires_grad else None     # d_y needs the weights alone
        ctx.save_for_backward(need_y, positions, offsets, weights)
        ctx.stride = stride
        return _combine(y, stride, positions, weights, shared, shared_stride, stream)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        y, positions, offsets, weights = ctx.saved_tensors
        want_y, want_w, want_s = (ctx.needs_input_grad[i] for i in (0, 4, 5))
        d_y = d_w = None
        if want_y or want_w:
            rows, stride = _grad_rows(g)
            n_tok, k = positions.shape
            H = rows.shape[1]
            c, st = on(rows.device, None)
            with c:
                d_y = rows.new_empty((n_tok * k, H)) if want_y else None
                d_w = torch.empty_like(weights) if want_w else None
                check(lib().moe_b200_combine_sorted_grad(
                    rows.data_ptr(), ELEM[rows.dtype], stride, None if y is None else y.data_ptr(), ctx.stride, n_tok, k, H,
                    positions.data_ptr(), offsets.data_ptr() + 4 * (offsets.shape[0] - 1), weights.data_ptr(),
                    None if d_y is None else d_y.data_ptr(), None if d_w is None else d_w.data_ptr(), st))
        return d_y, None, None, None, d_w, g if want_s else None, None, None


def _rows_of(t, name, n, order):
    stride = dense_rows(t, name)
    if t.dim() != 2 or t.shape[0] != n or t.shape[1] < 1:
        raise bad(f"{name} must be [{n}, H]")
    if t.device != order.device:
        raise bad(f"{name} and the order must be on one device")
    return stride


def gather_sorted(x, order, stream=None):
    """x f32 / f16 / bf16 [n_tok, H] -> [n_tok k, H]: the token of every sorted row,
    zeros behind the last one."""
    stride = _rows_of(x, "x", order.n_tok, order)
    if x.requires_grad and torch.is_grad_enabled():
        with on(x.device, stream)[0]:       # (the backward pass runs on the stream that is current here)
            return _Gather.apply(x, stride, *_tensors(order), stream)
    return _gather(x, stride, *_tensors(order), stream)


def dispatch_sorted(x, ids, n_experts, stream=None):
    """sort_by_expert and gather_sorted: (rows [n_tok k, H], order)."""
    dense_rows(x, "x")
    if isinstance(ids, torch.Tensor) and ids.dim() == 2 and (x.dim() != 2 or x.shape[0] != ids.shape[0] or x.device != ids.device):
        raise bad("x must be [n_tok, H] on the ids' device")
    order = ExpertOrder(ids, n_experts, stream)
    return gather_sorted(x, order, stream), order


def combine_sorted(y, order, weights, shared=None, stream=None):
    """y f32 / f16 / bf16 [n_tok k, H] in sorted order, weights f32 [n_tok, k] (a
    Router's) -> [n_tok, H]: the weighted sum of each token's rows in pick order, plus
    `shared` [n_tok, H] (the shared expert's) of y's type, in 32 bits, rounded once.
    Picks without a sorted row add nothing, whatever their weight is; y's rows behind the
    last sorted one are not read."""
    stride = _rows_of(y, "y", order.n_tok * order.k, order)
    if not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32 or weights.device != order.device or \
            tuple(weights.shape) != (order.n_tok, order.k) or not weights.is_contiguous():
        raise bad("weights must be contiguous f32 [n_tok, k] on the order's device")
    shared_stride = 0
    if shared is not None:
        shared_stride = _rows_of(shared, "shared", order.n_tok, order)
        if shared.dtype != y.dtype or shared.shape[1] != y.shape[1]:
            raise bad("shared must be [n_tok, H] of y's type")
    pos, offsets = _tensors(order)
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad or (shared is not None and shared.requires_grad)):
        with on(y.device, stream)[0]:
            return _Combine.apply(y, stride, pos, offsets, weights, shared, shared_stride, stream)
    return _combine(y, stride, pos, weights, shared, shared_stride, stream)


__all__ = ["ExpertOrder", "sort_by_expert", "gather_sorted", "dispatch_sorted", "combine_sorted"]
