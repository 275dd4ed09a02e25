"""Routing where 32-bit scores leave their range: sigmoid scores below the
smallest normal number, and sums of biases of the type's lowest value. Ids
against the 64-bit reference, exactly."""
import numpy as np
import pytest
import torch

import mx_ref as R

pytestmark = pytest.mark.gpu


def _check(pkg, cuda, logits, k, bias=None, **kw):
    lg = torch.from_numpy(np.asarray(logits, np.float32)).to(cuda)
    b = None if bias is None else torch.from_numpy(np.asarray(bias, np.float32)).to(cuda)
    ids, w = pkg.route_experts(lg, k, bias=b, **kw)
    rid, rw = R.route(lg.cpu().numpy(), k, bias=None if bias is None else np.asarray(bias, np.float32), **kw)
    np.testing.assert_array_equal(ids.cpu().numpy(), rid)
    np.testing.assert_allclose(w.cpu().numpy(), rw, rtol=5e-6, atol=2.0 ** -126)


@pytest.mark.parametrize("dtype_step", [0.0, 0.05])
def test_sigmoid_scores_that_underflow(pkg, cuda, dtype_step):
    """Logits from -86 to -104: the scores pass the smallest normal number, where a 32-bit quotient may return
    zero; a group's sum of two must not lose one of them."""
    rng = np.random.default_rng(0)
    kw = dict(score="sigmoid", n_group=2, topk_group=1, group_score="top2")
    _check(pkg, cuda, [[-86.70, -87.40, -87.0, -87.1], [-87.0, -87.1, -86.70, -87.40]], 2, **kw)
    l = -86 - 2.2 * rng.random((300, 64)) - dtype_step * rng.integers(0, 300, size=(300, 1))
    for group_score in ("max", "top2"):
        _check(pkg, cuda, l, 6, score="sigmoid", n_group=8, topk_group=3, group_score=group_score)
    _check(pkg, cuda, l, 6, score="sigmoid", bias=np.zeros(64))
    _check(pkg, cuda, l, 6, score="sigmoid", bias=1e-38 * rng.random(64), n_group=4, topk_group=2)


@pytest.mark.parametrize("score", ["sigmoid", "softmax", "softmax_topk"])
def test_biases_of_the_lowest_value(pkg, cuda, score):
    """Two biases of the type's lowest value add up to less than 32 bits hold; such a group is still ahead of
    one whose experts are all masked by -inf."""
    low = np.finfo(np.float32).min
    l = np.full((3, 8), -np.inf, np.float32)
    l[0, 0], l[0, 6:] = 0.5, [0.25, 0.5]
    l[1, 1], l[1, 4:6] = -0.5, [1.0, -1.0]
    l[2, 0], l[2, 4:] = 0.25, 0.0
    b = np.array([0, 0, 0, 0, low, low, low, low], np.float32)
    for k in (1, 2, 3, 4):
        _check(pkg, cuda, l, k, bias=b, score=score, n_group=4, topk_group=2, group_score="top2")
    both = np.where(np.isneginf(l), np.float32(low), l)          # logits masked by the lowest value, biases too
    for k in (2, 4):
        _check(pkg, cuda, both, k, bias=b, score=score, n_group=4, topk_group=2, group_score="top2")
        _check(pkg, cuda, both, k, bias=b, score=score)
