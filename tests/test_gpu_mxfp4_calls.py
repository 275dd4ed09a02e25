"""Calls of the MXFP4 operators that the documentation allows, off the main
path: short last runs of a row, waits that give up, streams, graphs, given
planes. Values against the 64-bit reference (mx_ref)."""
import numpy as np
import pytest
import torch

import mx_ref as R

pytestmark = pytest.mark.gpu


def _experts(rng, E, rows, K):
    return R.to_blocks(*R.quantize_plane(0.02 * rng.normal(size=(E, rows, K))))


def _weights(pkg, cuda, blocks, K):
    return pkg.MXFP4Weights(torch.from_numpy(blocks).to(cuda), K, blocks.shape[1])


def _ids(rng, n, k, E):
    return np.argsort(rng.normal(size=(n, E)), axis=1)[:, :k].astype(np.int32)


@pytest.mark.parametrize("planes", [1, 2])
@pytest.mark.parametrize("n,K", [(5500, 352), (4097, 608), (2400, 896)])   # 3, 5 and 7 K tiles
def test_long_prompt_with_an_odd_number_of_tiles(pkg, cuda, n, K, planes):
    """Rows whose tiles the halves of a warp share unevenly: one of them is at its row's last, single tile."""
    rng = np.random.default_rng(K)
    E, rows = 3, 40
    W = _experts(rng, E, rows, K)
    x = rng.normal(size=(n, K)).astype(np.float32)
    ids = rng.integers(0, E, size=(n, 1)).astype(np.int32)
    y = pkg.mxfp4_mul_mat_id(_weights(pkg, cuda, W, K), torch.from_numpy(x).to(cuda), torch.from_numpy(ids).to(cuda),
                             planes=planes).cpu().numpy()
    ref, mag = R.product(W, x, ids, planes)
    assert pkg.moe_cache.device_error() == 0
    assert (np.abs(y - ref) <= R.product_tol(mag, K, planes)).all()
