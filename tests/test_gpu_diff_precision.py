"""esp_attn_diff on the device: the weights' second 16 bits reach the product with V."""
import numpy as np
import pytest

from diff_precision import bound
from diff_utils import HD
from espetero_amd import abi
from oracle import binding as ob
from test_diff_precision import small_scores
from test_gpu_diff import Run

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16


def check(c, numbers, **plan):
    r = Run(c, **plan)
    want, tol = bound(c, numbers)
    got = ob.to_f32(r()[:, :c.H * 128], c.dtype)
    print(f"  of the bound: {np.max(np.abs(got - want) / tol):.3f}", flush=True)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,seqs", [((8, 4), [(40, 1), (17, 1)]), ((32, 4), [(30, 1)]), ((8, 4), [(20, 4), (0, 3)]), ((16, 4), [(33, 4)])])
def test_few_rows_hold_both_maps_weights_as_two_numbers(heads, seqs, dtype):
    c = small_scores(heads, dtype, seqs, 1.0)
    check(c, (2, 2))
    check(c, (2, 2), workgroups=4096)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,seqs", [((8, 4), [(20, 30)]), ((16, 4), [(11, 40), (33, 9)]), ((4, 4), [(0, 60)])])
def test_many_rows_hold_the_first_maps_weights_as_two_numbers(heads, seqs, dtype):
    check(small_scores(heads, dtype, seqs, 1.0), (2, 1))
    c = small_scores(heads, dtype, seqs, 0.0)                         # the first map alone
    check(c, (2, 1))
    check(c, (2, 1), workgroups=2048, cut_batch=True)


@pytest.mark.parametrize("cut", [False, True])
def test_many_rows_give_the_same_bits_again(cut):
    c = small_scores((16, 4), BF16, [(70, 90), (0, 200)], 1.0)
    r = Run(c, **(dict(workgroups=2048, cut_batch=True) if cut else {}))
    first = r()
    for _ in range(3):
        r.O.fill_(0x1234)
        assert (r() == first).all()


def alike(heads, dtype, seqs, weight):
    """Both maps of a pair are the same, which is where the operator takes most away: what the second one's weights lose is not small
    beside the difference."""
    c = small_scores(heads, dtype, seqs, 1.0)
    c.weight[:] = weight
    Q = c.Q[:, :c.H * HD].reshape(c.n_rows, c.H // 2, 2, HD)
    Q[:, :, 1] = Q[:, :, 0]
    pool = c.pool.reshape(c.n_blocks, c.Hkv // 2, 2, 2, c.bt * HD)
    pool[:, :, 1, 0] = pool[:, :, 0, 0]
    for K in c.K:
        K[:, 1::2] = K[:, ::2]
    return c


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("weight", [0.8, 1.0])
@pytest.mark.parametrize("heads,seqs", [((8, 4), [(33, 1), (20, 4)]), ((8, 4), [(20, 30)]), ((16, 4), [(11, 40), (33, 9)]), ((4, 4), [(0, 60)])])
def test_maps_that_are_alike_cancel_to_the_weights_own_bits(heads, seqs, weight, dtype):
    c = alike(heads, dtype, seqs, weight)
    check(c, (2, 2))
    check(c, (2, 2), workgroups=2048, cut_batch=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,seqs", [((8, 4), [(20, 30)]), ((16, 4), [(11, 40), (33, 9)]), ((4, 4), [(0, 60)])])
def test_many_rows_hold_both_maps_weights_as_two_numbers(heads, seqs, dtype):
    c = small_scores(heads, dtype, seqs, 1.0)
    check(c, (2, 2))
    check(c, (2, 2), workgroups=2048, cut_batch=True)
