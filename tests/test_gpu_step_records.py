"""The operators around a decode step where several passes share a record or a workspace, against the operators in float64."""
import numpy as np
import pytest
import torch

import test_gpu_lowrank as lowrank
from espetero_amd import abi, device

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16


def adapters(n, seed):
    return np.random.default_rng(seed).integers(-1, 2, n)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,rank", [(256, 8), (512, 40)])             # the small pass as one launch and as two
@pytest.mark.parametrize("first,second", [(300, 20), (20, 300)])
def test_two_lowrank_passes_of_one_record(first, second, D, rank, dtype):
    device.init(0)
    cases = [lowrank.Case(adapters(n, n), D, rank, lowrank.QKV, dtype, 2, seed=n) for n in (first, second)]
    for c in cases:
        c.A, c.B, c.scale = cases[0].A, cases[0].B, cases[0].scale
        c.prepare()
    p = device.lowrank_params(D, rank, lowrank.QKV, dtype, D, cases[0].y_ld, 2)
    for c in cases:
        c.lp = device.LowRankPass(p, c.adapter)
    for c in cases + cases[::-1]:                                    # in both orders
        c.dY.copy_(torch.from_numpy(c.Y))
        c.run()
        torch.cuda.synchronize()
        want, tol = c.expected()
        assert np.all(np.abs(c.dY.cpu().numpy() - want) <= tol)
