"""The operators around a decode step where several passes share a record or a workspace, against the operators in float64."""
import numpy as np
import pytest
import torch

import test_gpu_lowrank as lowrank
from espetero_amd import abi, device, synth
from oracle import binding as ob

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


def far_apart(rank, n, apart, dtype):
    """A row's intermediates lie `apart` powers of two below its first, which half of the columns of B leave out; Y is zero."""
    c = lowrank.Case([0] * n, 8, rank, lowrank.QKV, dtype, 1, seed=apart)
    small = ob.to_f32(c.A, dtype) * np.float32(2.0 ** -(apart // 2))
    small[:, ::rank] *= np.float32(2.0 ** apart)
    c.A = synth._bits(small, dtype)
    B = c.B.reshape(-1, rank)
    B[::2, 0] = 0
    c.Y[:] = 0
    return c


def far_apart_bound(c):
    """As lowrank.Case.expected, with each intermediate's own size where that takes the row's largest: two fp16 numbers hold one to
    2^-23 of itself, and to 2^-39 of the row's largest, which is 2^14 or more when half a step of the smallest numbers is 2^-25. Three
    bf16 numbers hold it to 2^-24."""
    f = lambda x: ob.to_f32(x, c.dtype).astype(np.float64)  # noqa: E731
    X, A, B, scale, at = f(c.X), f(c.A)[0], f(c.B)[0], float(c.scale[0]), 0
    Y, tol = np.zeros(c.Y.shape), np.zeros(c.Y.shape)
    for s, (off, w) in enumerate(c.slices):
        As, Bs = A[s * c.rank:(s + 1) * c.rank], B[at:at + w]
        low, mag = X @ As.T, np.abs(X) @ np.abs(As).T
        e = (c.D + 16) * 2.0 ** -24 * mag + 2.0 ** -23 * np.abs(low) + 2.0 ** -39 * np.abs(low).max(1, keepdims=True)
        size = np.abs(low) @ np.abs(Bs).T
        Y[:, off:off + w] = scale * (low @ Bs.T)
        tol[:, off:off + w] = scale * (e @ np.abs(Bs).T + (4 * c.rank * 2.0 ** -24 + 2.0 ** -22) * size)
        at += w
    return Y, tol


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("apart", [8, 16])
@pytest.mark.parametrize("rank,n", [(8, 5), (24, 3), (40, 20), (16, 150), (128, 140)])   # one launch, two, and tiles of 64 rows
def test_small_intermediates_beside_a_large_one_keep_their_bits(rank, n, apart, dtype):
    c = far_apart(rank, n, apart, dtype).prepare()
    c.run()
    torch.cuda.synchronize()
    want, tol = far_apart_bound(c)
    err = np.abs(c.dY.cpu().numpy() - want)
    print(f"  of the bound: {np.max(err / tol):.3f}", flush=True)
    assert np.all(err <= tol)
