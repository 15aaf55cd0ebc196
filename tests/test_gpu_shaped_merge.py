"""esp_attn_shaped on the device: infinite values in passes whose tiles are split, which their merge has to leave infinite."""
import numpy as np
import pytest

from shaped_utils import ShapedCase
from test_gpu_shaped import Run, dev
from espetero_amd import abi
from oracle import binding as ob

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16


def run(c, places, **plan):
    """(clean, got): outputs [rows][H][hd] as they are, and with infinities in the dims of the keys of `places`, {key: (dim of +inf, dim of -inf)}, in KV
    head 0."""
    r = Run(c, **plan)
    assert r.parts and any(int(n) % 4 for n in r.jobs["nparts"]), "no tile of an odd number of parts"
    clean = r().reshape(c.n_rows, c.H, c.hd)
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * c.hd)
    for j, (plus, minus) in places.items():
        V = pool[c.block_list[j // c.bt], 0, 1].reshape(c.bt // 16, c.hd, 16)
        V[j % c.bt // 16, plus, j % 16] = 0x7C00 if c.dtype == F16 else 0x7F80
        V[j % c.bt // 16, minus, j % 16] = 0xFC00 if c.dtype == F16 else 0xFF80
    r.pool = dev(pool.reshape(-1))
    r.O.fill_(0x1234)
    return clean, r().reshape(c.n_rows, c.H, c.hd)


def infinite_in_every_part(heads, hd, P, M, dtype, **plan):
    c = ShapedCase(*heads, hd, dtype, 16, [(P, M)], sharp=0.25, seed=5)
    places = {j: (2 * i, 2 * i + 1) for i, j in enumerate(range(5, P, max(30, P // (hd // 2) + 1)))}
    clean, bits = run(c, places, **plan)
    got, G, n = ob.to_f32(bits, dtype), c.H // c.Hkv, 2 * len(places)
    assert (got[:, :G, 0:n:2] == np.inf).all() and (got[:, :G, 1:n:2] == -np.inf).all()
    assert np.isfinite(got[:, :G, n:]).all() and (bits[:, G:] == clean[:, G:]).all()


# Merges of four wavefronts an output (few outputs, many parts) and of one (many outputs).
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,hd,P,M", [((4, 4), 128, 333, 60), ((32, 8), 128, 333, 200), ((16, 1), 256, 500, 20), ((4, 4), 128, 600, 40)])
def test_many_rows(heads, hd, P, M, dtype):
    infinite_in_every_part(heads, hd, P, M, dtype, workgroups=2048, cut_batch=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,hd,P,M,workgroups", [((8, 4), 128, 700, 3, 64), ((32, 1), 256, 900, 4, 64), ((4, 4), 128, 600, 2, 24), ((32, 8), 128, 1500, 4, 40),
                                                     ((8, 4), 128, 700, 1, 64)])
def test_few_rows(heads, hd, P, M, workgroups, dtype):
    infinite_in_every_part(heads, hd, P, M, dtype, workgroups=workgroups)


@pytest.mark.parametrize("M,dtype", [(2, F16), (2, BF16), (40, BF16)])
def test_a_part_that_weighs_nothing_is_still_infinite(M, dtype):
    """A bias that leaves the part of an early key 2^-200 of the largest weight. (One row does not see the key.)"""
    c = ShapedCase(4, 4, 128, dtype, 16, [(600, M)], bias=True, spans=[[(0, 0)] * (M - 1) + [(9, 0)]], seed=6)
    c.slopes[:] = 0.25
    clean, bits = run(c, {8: (3, 60)}, workgroups=4096, cut_batch=True)
    got = ob.to_f32(bits, dtype)
    assert (got[:-1, 0, 3] == np.inf).all() and (got[:-1, 0, 60] == -np.inf).all()
    assert (bits[-1] == clean[-1]).all() and (bits[:, 1:] == clean[:, 1:]).all()
