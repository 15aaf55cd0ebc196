"""Linear attention's sequences in segments of any number of chunks, planned by hand: what a plan of any device may hold."""
import ctypes as C

import numpy as np
import pytest
import torch

from espetero_amd import abi, device
from linear_utils import LinearCase
from oracle import binding as ob
from test_gpu_linear import BF16, F16, Run, check

pytestmark = pytest.mark.gpu


def cut(r, each):
    """Run r's pass with each sequence in segments of `each` chunks."""
    c, tiles, parts = r.case, [], 0
    for base, rows, src, dst in c.records.tolist():
        n = max(1, -(-rows // (64 * each)))
        for k in range(n):
            at, end = 64 * each * k, min(rows, 64 * each * (k + 1))
            tiles.append((base + at, end - at, src, dst if k + 1 == n else -1, parts if n > 1 else -1, k, n - 1 - k, 0))
        parts += n if n > 1 else 0
    t = np.array(tiles, abi.LINEAR_TILE_DT)
    device.validate_linear(r.lp.params, t, 0, parts, c.n_rows)
    r.lp.tiles, r.lp.n_tiles, r.lp.n_few, r.lp.n_parts = device.to_dev(t), len(t), 0, parts
    nbytes = abi.attn_lib().esp_linear_workspace_bytes(C.byref(r.lp.params), parts)
    r.lp.workspace = torch.full((max(nbytes, 16),), 0xff, dtype=torch.uint8, device="cuda")   # NaN: nothing is read that was not written
    return r


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (128, 64), (64, 192)])
@pytest.mark.parametrize("each", [1, 2, 5])
def test_any_segments(each, dims, dtype):
    c = LinearCase(3, 1, *dims, dtype, [(400, 0, 0), (65, -1, 1), (321, 2, 3), (64, 4, 4), (192, 5, -1)], n_states=6, seed=31, row_decay=each == 2)
    check(c, cut(Run(c), each)())


@pytest.mark.parametrize("dims", [(64, 64), (128, 128)])
def test_more_segments_than_lanes(dims):
    """135 and 130 segments of a chunk each, whose decays a wavefront sums up 64 at a time."""
    for dtype, rows in ((F16, 64 * 135 - 3), (BF16, 64 * 130)):
        c = LinearCase(1, 1, *dims, dtype, [(rows, 0, 0)], seed=38, decay=-0.002)
        check(c, cut(Run(c), 1)())


@pytest.mark.parametrize("decay", [0.0, -1e-4, -3.0, -60.0, -200.0, float("-inf"), 1.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decays_across_segments(decay, dtype):
    c = LinearCase(2, 2, 64, 64, dtype, [(300, 0, 0), (200, 1, 1)], seed=32, decay=decay)
    check(c, cut(Run(c), 1)())
    check(c, cut(Run(c), 2)())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_row_that_forgets_everything_across_segments(dtype):
    c = LinearCase(2, 2, 64, 64, dtype, [(500, 0, 0), (130, 1, 1)], seed=33, row_decay=True)
    c.decay[[0, 63, 64, 127, 130, 191, 192, 499]] = -np.inf
    c.decay[200:260] = -100.0
    c.decay[300:430] = 0.0
    check(c, cut(Run(c), 1)())
    check(c, cut(Run(c), 3)())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("what", ["Q", "K", "V"])
def test_what_is_not_finite_stays_behind_its_row_across_segments(what, dtype):
    rows, r0 = 330, 140
    c = LinearCase(2, 2, 64, 64, dtype, [(rows, 0, 0), (rows, 1, 1)], seed=34)
    clean, _ = cut(Run(c), 1)()
    inf = 0x7C00 if dtype == F16 else 0x7F80
    for bad in (inf, inf | 0x8000, inf | 1):
        x = getattr(c, what).copy()
        getattr(c, what)[r0, 5] = bad
        bits, states = cut(Run(c), 1)()
        setattr(c, what, x)
        assert (bits[:r0] == clean[:r0]).all(), (what, bad)
        assert (bits[rows:] == clean[rows:]).all() and (bits[:, 64:] == clean[:, 64:]).all()
        if what == "V":
            rest = np.arange(64) != 5
            assert (bits[:rows, :64][:, rest] == clean[:rows, :64][:, rest]).all()
            assert not np.isfinite(ob.to_f32(bits[r0:rows, 5], dtype)).any()                     # its own column, from its row on
            assert not np.isfinite(states[0, 0, :, 5]).any() and np.isfinite(states[0, 0][:, rest]).all()
        if what == "K":
            assert not np.isfinite(ob.to_f32(bits[r0:rows, :64], dtype)).any()
        if what == "Q":
            assert not np.isfinite(ob.to_f32(bits[r0, :64], dtype)).any() and (bits[r0 + 1:] == clean[r0 + 1:]).all()


def test_an_infinite_state_across_segments():
    c = LinearCase(1, 1, 64, 64, BF16, [(200, 0, 0)], seed=35)
    clean, _ = cut(Run(c), 1)()
    c.states[0, 0, 9, 5] = np.inf
    bits, states = cut(Run(c), 1)()
    rest = np.arange(64) != 5
    assert not np.isfinite(ob.to_f32(bits[:, 5], BF16)).any() and not np.isfinite(states[0, 0, 9, 5])
    assert (bits[:, rest] == clean[:, rest]).all() and np.isfinite(states[0, 0][:, rest]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_states_of_few_sizes_across_segments(dtype):
    """Segments whose states differ by many powers of two: what a segment leaves is not lost beside what is in front of it, nor the other way round."""
    for first, second in ((1.0, 2.0 ** -9), (2.0 ** -9, 1.0)):
        c = LinearCase(1, 1, 64, 64, dtype, [(256, -1, 0)], seed=36, decay=-0.01)
        V = ob.to_f32(c.V, dtype).reshape(256, -1)
        V[:128] *= first
        V[128:] *= second
        c.V = ob.from_f32(V.reshape(-1), dtype).reshape(256, -1)
        check(c, cut(Run(c), 1)())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,r0", [(7, 3), (300, 37), (300, 64), (300, 200)])
def test_a_decay_that_is_no_number_stays_behind_its_row(rows, r0, dtype):
    """NaN as a row's log decay: that row and those behind it, of that head, have no value; the others keep their bits."""
    c = LinearCase(2, 2, 64, 64, dtype, [(rows, 0, 0), (rows, 1, 1)], seed=37, row_decay=True)
    run = (lambda: Run(c)()) if rows < 9 else (lambda: cut(Run(c), 2)())
    clean, clean_states = run()
    c.decay[r0, 1] = np.nan
    bits, states = run()
    assert (bits[:r0] == clean[:r0]).all() and (bits[rows:] == clean[rows:]).all() and (bits[:, :64] == clean[:, :64]).all()
    assert np.isnan(ob.to_f32(bits[r0:rows, 64:], dtype)).all() and np.isnan(states[0, 1]).all()
    assert (states[0, 0] == clean_states[0, 0]).all() and (states[1] == clean_states[1]).all()
