"""Routing tokens to experts with the scores of current MoE routers
(moe_b200_route_experts in include/moe_cache_b200.h)."""
import ctypes

import torch

from ._call import ELEM, bad, dense_rows, given, keep, on
from ._lib import MoeRouter, check, lib

SCORES = {"softmax": 0, "sigmoid": 1, "softmax_topk": 2}
GROUP_SCORES = {"max": 0, "top2": 1}


class Router:
    """How a layer routes: `score` "softmax" (over all experts), "sigmoid" or
    "softmax_topk" (over the picks); `bias` f32 [n_experts] that only the choice
    sees; `n_group` groups of consecutive experts, of which the `topk_group`
    best stay (by their largest selection score, "max", or the sum of their two
    largest, "top2"); `norm_w` divides the weights by their sum, `scale`
    multiplies them."""

    def __init__(self, k, score="softmax", bias=None, n_group=1, topk_group=1, group_score="top2", norm_w=False, scale=1.0):
        if score not in SCORES:
            raise bad(f"score must be one of {sorted(SCORES)}")
        if group_score not in GROUP_SCORES:
            raise bad(f"group_score must be one of {sorted(GROUP_SCORES)}")
        if bias is not None and not (isinstance(bias, torch.Tensor) and bias.is_cuda and bias.dtype == torch.float32 and
                                     bias.dim() == 1 and bias.is_contiguous()):
            raise bad("bias must be a contiguous f32 CUDA vector")
        self.k, self._bias = k, bias
        self.desc = MoeRouter(SCORES[score], n_group, topk_group, GROUP_SCORES[group_score], norm_w, scale)
        self.ref = ctypes.byref(self.desc)

    @property
    def bias(self):
        """The bias (written in place, it takes effect from the next call on)."""
        return self._bias

    def __call__(self, logits, ids=None, weights=None, stream=None):
        """logits f32 / f16 / bf16 [n_tok, E] -> (ids i32 [n_tok, k], weights f32 [n_tok, k]).
        With `stream` a torch.cuda.Stream the tensors may be dropped right behind the
        call, with a raw handle the caller keeps them until the stream has run it."""
        stride = dense_rows(logits, "logits")
        if logits.dim() != 2:
            raise bad("logits must be [n_tok, n_experts]")
        n_tok, E = logits.shape
        k, dev, bias = self.k, logits.device, self._bias
        if bias is not None and (bias.device != dev or bias.shape[0] != E):
            raise bad("bias must be f32 [n_experts] on the logits' device")
        ctx, st = on(dev, stream)
        with ctx:
            ids = logits.new_empty((n_tok, k), dtype=torch.int32) if ids is None else \
                given(ids, "ids", torch.int32, (n_tok, k), dev)
            weights = logits.new_empty((n_tok, k), dtype=torch.float32) if weights is None else \
                given(weights, "weights", torch.float32, (n_tok, k), dev)
            check(lib().moe_b200_route_experts(self.ref, logits.data_ptr(), ELEM[logits.dtype], stride,
                                               None if bias is None else bias.data_ptr(), n_tok, E, k,
                                               ids.data_ptr(), weights.data_ptr(), st))
        keep(stream, logits, bias, ids, weights)
        return ids, weights


def route_experts(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_score="top2", norm_w=False,
                  scale=1.0, ids=None, weights=None, stream=None):
    """One routing call (see Router): (ids i32 [n_tok, k], weights f32 [n_tok, k])."""
    return Router(k, score, bias, n_group, topk_group, group_score, norm_w, scale)(logits, ids, weights, stream)


__all__ = ["Router", "route_experts"]
