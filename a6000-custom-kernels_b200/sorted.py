"""Tokens sorted by expert and back (include/moe_cache_b200.h): the order of the
picks by expert, the tokens' rows in that order, and the weighted sum of such rows
back into the tokens, with gradients -- for experts that run outside this library.

    rows, order = dispatch_sorted(x, ids, n_experts)     # rows of expert e: order.offsets[e] to [e + 1]
    out = combine_sorted(experts(rows, order.offsets), order, weights)

`stream` is a torch.cuda.Stream, a raw handle, or None for the device's current
stream; outputs are allocated on it. With a torch.cuda.Stream the inputs may be
dropped right behind the call, with a raw handle the caller keeps them until the
stream has run it. gather_sorted, dispatch_sorted and combine_sorted are
differentiable once (in x, y, weights and shared; forward-mode derivatives are refused);
their backward pass runs on the stream of the call. A pass may be captured into a graph
while no autograd graph of the same leaves that was made on another stream is alive
(autograd would make the capture wait for that stream): next to such a graph of these
calls a call is refused, whether it takes the leaves or what was computed from them.
Graphs of other operations only are the caller's to drop.
"""
import threading
import weakref

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._call import ELEM, bad, dense_rows, keep, no_tangents, on
from ._lib import check, lib


class ExpertOrder:
    """The picks of n_tok tokens by expert: `rows` i32 [n_tok k], the entry t k + j of
    each sorted row, and `experts`, its expert (-1 behind the last row); `positions`
    i32 [n_tok, k], the sorted row of a pick or -1; `offsets` i32 [n_experts + 1], the
    first sorted row of each expert, then their number."""

    def __init__(self, ids, n_experts):
        """(dispatch_sorted and sort_by_expert make orders)"""
        if not (isinstance(ids, torch.Tensor) and ids.is_cuda and ids.dtype == torch.int32 and ids.dim() == 2):
            raise bad("ids must be an i32 CUDA tensor [n_tok, k]")
        n_tok, k = ids.shape
        self._stride = k
        if not ids.is_contiguous() and n_tok > 0:
            self._stride = ids.stride(0) if n_tok > 1 else k
            if (ids.stride(1) != 1 and k > 1) or self._stride < k:
                raise bad("ids' rows must be dense and must not overlap in memory")
        if k < 1 or n_experts < 1:
            raise bad("need k >= 1 and n_experts >= 1")
        self.n_tok, self.k, self.n_experts, self.device = n_tok, k, n_experts, ids.device
        self._views = None

    def _allocate(self, ids):
        """Memory for the order (rows, positions, experts, offsets behind one another) and their addresses."""
        n = self.n_tok * self.k
        self._buf = ids.new_empty(3 * n + self.n_experts + 1)
        at = self._buf.data_ptr()
        self._at = at, at + 4 * n, at + 8 * n, at + 12 * n
        return self._at

    def _view(self, i):
        if self._views is None:
            n = self.n_tok * self.k
            self._views = self._buf.split([n, n, n, self.n_experts + 1])
        return self._views[i]

    @property
    def rows(self):
        return self._view(0)

    @property
    def positions(self):
        return self._view(1).view(self.n_tok, self.k)

    @property
    def experts(self):
        return self._view(2)

    @property
    def offsets(self):
        return self._view(3)


def sort_by_expert(ids, n_experts, stream=None):
    """ids i32 [n_tok, k] (a Router's; -1: an empty slot) -> the ExpertOrder of its
    picks: by expert, and within one in the order of (token, pick)."""
    order = ExpertOrder(ids, n_experts)
    ctx, st = on(ids.device, stream)
    with ctx:
        check(lib().moe_b200_sort_by_expert(ids.data_ptr(), order._stride, order.n_tok, order.k, n_experts, *order._allocate(ids), st))
    keep(stream, ids, order._buf)
    return order


# The row calls take the order's memory (_buf) and its sizes: positions start n_tok k words in, the number of
# sorted rows is its last word.
def _gather(x, stride, buf, n_tok, k, stream):
    n, H = n_tok * k, x.shape[1]
    ctx, st = on(x.device, stream)
    with ctx:
        out = x.new_empty((n, H))
        at = buf.data_ptr()
        check(lib().moe_b200_gather_sorted(x.data_ptr(), ELEM[x.dtype], stride, n_tok, k, H, at + 4 * n,
                                           at + 4 * (buf.shape[0] - 1), out.data_ptr(), st))
    if stream is not None:
        keep(stream, x, buf, out)
    return out


def _combine(y, stride, buf, n_tok, k, weights, shared, shared_stride, stream):
    H = y.shape[1]
    ctx, st = on(y.device, stream)
    with ctx:
        out = y.new_empty((n_tok, H))
        check(lib().moe_b200_combine_sorted(y.data_ptr(), ELEM[y.dtype], stride, n_tok, k, H, buf.data_ptr() + 4 * n_tok * k,
                                            None if weights is None else weights.data_ptr(),
                                            None if shared is None else shared.data_ptr(), shared_stride, out.data_ptr(), st))
    if stream is not None:
        keep(stream, y, buf, weights, shared, out)
    return out


# ---- gradients -----------------------------------------------------------------

_alive, _alive_lock = weakref.WeakSet(), threading.Lock()      # autograd nodes of the calls below; `made`: their stream


def _remember(node):
    with _alive_lock:
        _alive.add(node)


def _leaves(tensors, nodes):
    """The leaves (by id; their graphs keep them) that gradients of these tensors, and those that pass these nodes, reach."""
    leaves = {id(t) for t in tensors if t is not None and t.requires_grad and t.is_leaf}
    todo = [*nodes, *(t.grad_fn for t in tensors if t is not None and t.grad_fn is not None)]
    seen = set(todo)
    while todo:
        for node, _ in todo.pop().next_functions:
            if node is None or node in seen:
                continue
            seen.add(node)
            if not node.next_functions and hasattr(node, "variable"):      # where a leaf's gradient is added up
                leaves.add(id(node.variable))
            else:
                todo.append(node)
    return leaves


def _check_capture(st, *tensors):
    if torch.cuda.is_current_stream_capturing():
        with _alive_lock:
            others = [node for node in _alive if node.made != st]
        meet = others and not _leaves(tensors, ()).isdisjoint(_leaves((), others))
        del others      # (the error's traceback would keep them)
        if meet:
            raise bad("an autograd graph of the same leaves, made on another stream, is alive: drop it before the capture")


def _grad_rows(g):
    """A gradient as rows that the calls take (autograd may hand over an expanded one) and their stride."""
    H = g.shape[1]
    if not g.is_contiguous() and (g.stride(1) != 1 or g.stride(0) < H):
        g = g.contiguous()
    return g, max(g.stride(0), H)


def _differentiable_once(backward):
    """once_differentiable where a graph of the gradients is being made, the plain call (faster) where it is not."""
    checked = once_differentiable(backward)
    return lambda ctx, *g: (checked if torch.is_grad_enabled() else backward)(ctx, *g)


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, buf, n_tok, k, made, rows):
        ctx.save_for_backward(buf)
        ctx.call, ctx.made = (n_tok, k), made
        _remember(ctx)
        return rows()

    @staticmethod
    @_differentiable_once
    def backward(ctx, g):
        g, stride = _grad_rows(g)
        return _combine(g, stride, ctx.saved_tensors[0], *ctx.call, None, None, 0, None), None, None, None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, stride, buf, n_tok, k, weights, shared, shared_stride, made, stream):
        ctx.save_for_backward(y if weights.requires_grad else None, buf, weights)     # d_y needs the weights alone
        ctx.call, ctx.made = (stride, n_tok, k), made
        _remember(ctx)
        return _combine(y, stride, buf, n_tok, k, weights, shared, shared_stride, stream)

    @staticmethod
    @_differentiable_once
    def backward(ctx, g):
        y, buf, weights = ctx.saved_tensors
        want = ctx.needs_input_grad
        d_y = d_w = None
        if want[0] or want[5]:
            rows, stride = _grad_rows(g)
            y_stride, n_tok, k = ctx.call
            n, H = n_tok * k, rows.shape[1]
            c, st = on(rows.device, None)
            with c:
                d_y = rows.new_empty((n, H)) if want[0] else None
                d_w = torch.empty_like(weights) if want[5] else None
                at = buf.data_ptr()
                check(lib().moe_b200_combine_sorted_grad(
                    rows.data_ptr(), ELEM[rows.dtype], stride, None if y is None else y.data_ptr(), y_stride, n_tok, k, H,
                    at + 4 * n, at + 4 * (buf.shape[0] - 1), weights.data_ptr(), None if d_y is None else d_y.data_ptr(),
                    None if d_w is None else d_w.data_ptr(), st))
        return d_y, None, None, None, None, d_w, g if want[6] else None, None, None, None


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
    if forward_ad._current_level >= 0:
        no_tangents(x)
    if not (x.requires_grad and torch.is_grad_enabled()):
        return _gather(x, stride, order._buf, order.n_tok, order.k, stream)
    ctx, st = on(x.device, stream)
    with ctx:       # (the backward pass runs on the stream that is current here)
        _check_capture(st, x)
        return _Gather.apply(x, order._buf, order.n_tok, order.k, st,
                             lambda: _gather(x, stride, order._buf, order.n_tok, order.k, stream))


def dispatch_sorted(x, ids, n_experts, stream=None):
    """sort_by_expert and gather_sorted in one call: (rows [n_tok k, H], order)."""
    order = ExpertOrder(ids, n_experts)
    stride = _rows_of(x, "x", order.n_tok, order)
    if forward_ad._current_level >= 0:
        no_tangents(x)
    n_tok, k, H = order.n_tok, order.k, x.shape[1]
    ctx, st = on(x.device, stream)

    def rows():
        out = x.new_empty((n_tok * k, H))
        check(lib().moe_b200_dispatch_sorted(x.data_ptr(), ELEM[x.dtype], stride, H, ids.data_ptr(), order._stride, n_tok, k,
                                             n_experts, *at, out.data_ptr(), st))
        return out
    with ctx:
        if x.requires_grad and torch.is_grad_enabled():
            _check_capture(st, x)
            at = order._allocate(ids)
            out = _Gather.apply(x, order._buf, n_tok, k, st, rows)
        else:
            at = order._allocate(ids)
            out = rows()
    if stream is not None:
        keep(stream, x, ids, order._buf, out)
    return out, order


def combine_sorted(y, order, weights, shared=None, stream=None):
    """y f32 / f16 / bf16 [n_tok k, H] in sorted order, weights f32 [n_tok, k] (a
    Router's) -> [n_tok, H]: the weighted sum of each token's rows in pick order, plus
    `shared` [n_tok, H] (the shared expert's) of y's type, in 32 bits, rounded once.
    Picks without a sorted row add nothing, whatever their weight is; y's rows behind the
    last sorted one are not read."""
    n_tok, k = order.n_tok, order.k
    stride = _rows_of(y, "y", n_tok * k, order)
    if not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32 or weights.device != order.device or \
            weights.shape != (n_tok, k) or not weights.is_contiguous():
        raise bad("weights must be contiguous f32 [n_tok, k] on the order's device")
    shared_stride, grad = 0, y.requires_grad or weights.requires_grad
    if shared is not None:
        shared_stride = _rows_of(shared, "shared", n_tok, order)
        if shared.dtype != y.dtype or shared.shape[1] != y.shape[1]:
            raise bad("shared must be [n_tok, H] of y's type")
        grad = grad or shared.requires_grad
    if forward_ad._current_level >= 0:
        no_tangents(y, weights, shared)
    if not (grad and torch.is_grad_enabled()):
        return _combine(y, stride, order._buf, n_tok, k, weights, shared, shared_stride, stream)
    ctx, st = on(y.device, stream)
    with ctx:
        _check_capture(st, y, weights, shared)
        return _Combine.apply(y, stride, order._buf, n_tok, k, weights, shared, shared_stride, st, stream)


__all__ = ["ExpertOrder", "sort_by_expert", "gather_sorted", "dispatch_sorted", "combine_sorted"]
