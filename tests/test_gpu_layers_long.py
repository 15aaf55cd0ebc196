"""Linear attention and attention with shaped scores on the device at the lengths they are for, and at the border between linear attention's two
kernels."""
import numpy as np
import pytest

from linear_utils import LinearCase
from shaped_precision import bound
from shaped_utils import ShapedCase, documents
from test_gpu_linear import Run as LinearRun
from test_gpu_linear import check as linear_check
from test_gpu_shaped import Run
from espetero_amd import abi, synth
from oracle import binding as ob

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16


def check(c, rows, shift, **plan):
    r = Run(c, **plan)
    want, tol, which = bound(c, shift, rows)
    got = ob.to_f32(r()[which][:, :c.H * c.hd], c.dtype).astype(np.float64).reshape(want.shape)
    print(f"  of the bound: {np.max(np.abs(got - want) / tol):.3f}", flush=True)
    assert np.all(np.abs(got - want) <= tol)


SHAPES = [(0.0, False), (20.0, False), (0.0, True), (30.0, True)]


@pytest.mark.parametrize("cap,bias", SHAPES)
@pytest.mark.parametrize("heads,hd,dtype,P,M,window", [((8, 2), 128, BF16, 9000, 130, 0), ((4, 2), 256, F16, 9100, 70, 0), ((4, 4), 128, F16, 16000, 40, 0),
                                                       ((8, 2), 128, F16, 12345, 60, 5000)])
def test_many_rows_behind_a_long_cache(heads, hd, dtype, P, M, window, cap, bias):
    c = ShapedCase(*heads, hd, dtype, 16, [(P, M)], cap=cap, bias=bias, window=window, seed=P)
    rows = sorted({0, 1, M // 2, M - 1})
    check(c, rows, 7, workgroups=1)                                    # whole tiles
    check(c, rows, 7)


@pytest.mark.parametrize("cap,bias", SHAPES)
@pytest.mark.parametrize("heads,hd,dtype,M", [((8, 2), 128, F16, 1), ((8, 2), 128, BF16, 7), ((4, 2), 256, BF16, 3)])
def test_few_rows_behind_a_long_cache(heads, hd, dtype, M, cap, bias):
    c = ShapedCase(*heads, hd, dtype, 16, [(20000, M)], cap=cap, bias=bias, seed=M)
    check(c, {0, M - 1}, 15, workgroups=1)
    check(c, {0, M - 1}, 15)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,cap", [(128, 0.0), (128, 60.0), (256, 0.0)])
@pytest.mark.parametrize("starts", [[0], [0, 3000], [0, 100, 9030]])
def test_far_keys_move_a_reference_late(starts, hd, cap, dtype):
    """Keys are larger the further back they lie, so that the rows' largest scores come last, again and again; documents and a prefix of half of each."""
    P, M = 9000, 70
    c = ShapedCase(4, 2, hd, dtype, 16, [(P, M)], cap=cap, spans=[documents(P, M, starts, 50)] if len(starts) > 1 else None, seed=9)
    grow = np.linspace(6.0, 0.2, P + M, dtype=np.float32)[:, None, None]
    c.K[0][:] = synth._bits(ob.to_f32(c.K[0], dtype) * grow, dtype)
    pool = c.pool.reshape(c.n_blocks, 2, 2, 16 * hd)
    for j in range(P + M):
        pool[c.block_list[j // 16], :, 0].reshape(2, 16, hd)[:, j % 16] = c.K[0][j]
    check(c, [0, 33, M - 1], 7, workgroups=1)
    check(c, [0, 33, M - 1], 7)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("row_decay", [False, True])
@pytest.mark.parametrize("workgroups", [1, 512])
def test_linear_attention_of_a_long_document(workgroups, row_decay, dtype):
    c = LinearCase(4, 2, 64, 128, dtype, [(16000, 0, 1)], n_states=3, row_decay=row_decay, seed=16)
    r = LinearRun(c, workgroups=workgroups)
    linear_check(c, r())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 128), (128, 512)])
@pytest.mark.parametrize("row_decay", [False, True])
def test_linear_attention_of_seven_to_nine_rows(row_decay, dk, dv, dtype):
    c = LinearCase(4, 2, dk, dv, dtype, [(8, 0, 0), (9, 1, 2), (7, -1, 3), (8, 4, -1), (8, -1, 5), (9, 6, 6)], n_states=8, row_decay=row_decay, seed=dv)
    r = LinearRun(c)
    assert r.lp.n_few == 4 and r.lp.n_tiles == 6
    linear_check(c, r())
