"""The bound that the device's outputs are held to where weights are two 16-bit numbers (tests/test_gpu_diff_precision.py): weights of one
number do not stay within it."""
import numpy as np
import pytest

from diff_precision import bound, with_weights_of
from diff_utils import DiffCase
from espetero_amd import abi


def small_scores(heads, dtype, seqs, second):
    """Even weights, whose rounding shows and whose scores' does not. second: of the second map's weight."""
    c = DiffCase(*heads, dtype, 16, seqs, seed=21, norm=False, sharp=0.02)
    c.weight *= np.float32(second)
    return c


@pytest.mark.parametrize("dtype", [abi.ESP_F16, abi.ESP_BF16])
def test_the_bound_tells_one_number_from_two(dtype):
    c = small_scores((8, 4), dtype, [(33, 1), (20, 4)], 1.0)
    want, tol = bound(c, (2, 2))
    off = lambda k: np.abs(with_weights_of(c, k) - want) > tol  # noqa: E731
    assert not off((2, 2)).any() and not off((3, 3)).any()
    assert off((1, 2)).mean() > 0.01 and off((2, 1)).mean() > 0.01
    want, tol = bound(c, (2, 1))
    assert not off((2, 1)).any()
    c = small_scores((8, 4), dtype, [(33, 1), (20, 4)], 0.0)         # without the second map its bound adds nothing
    want, tol = bound(c, (2, 1))
    assert not off((2, 1)).any() and off((1, 1)).mean() > 0.01
