"""What the passes of the operators around a decode step keep of a caller's parameter record, host-side checks of their records and the
sizes of their workspaces. No GPU: records are built in host memory and every call is refused."""
import ctypes as C

import numpy as np
import pytest
import torch

from espetero_amd import abi, device, host, synth


# ---- one record, several passes
@pytest.mark.parametrize("first,second", [(200, 20), (20, 200), (1000, 4)])
def test_lowrank_passes_of_one_record_keep_their_own_tiles(first, second):
    """A prompt's pass and a decode step's pass of one layer: the record is the layer's, the tiles are each pass's own."""
    p = device.lowrank_params(256, 16, [(0, 64), (64, 32)], abi.ESP_F16, 256, 96, 2)
    before = bytes(p)
    a = device.LowRankPass(p, [0] * first, device="cpu")
    of_a = bytes(a.params)
    b = device.LowRankPass(p, [1] * second, device="cpu")
    assert bytes(p) == before and bytes(a.params) == of_a
    for x, n in ((a, first), (b, second)):
        assert x.params.rows_per_tile == (16 if n <= 128 else 64)
        tiles = x.tiles.numpy().view(abi.LOWRANK_TILE_DT)
        assert tiles["count"].max() == min(n, x.params.rows_per_tile) and tiles["count"].sum() == n
    p.D = 8                                                          # nor does a later change of the record reach them
    assert a.params.D == b.params.D == 256


def test_a_diff_pass_refuses_to_run_with_other_tiles_than_its_own():
    """The record stays the caller's, who may move its pool's region; the tiles are planned for one rows_per_tile."""
    p = synth.make_params(8, 4, 128, abi.ESP_F16, 16, rows_per_tile=1)
    none = torch.zeros(4)
    passes = []
    for M in (100, 1):
        p.rows_per_tile = device.attn_diff_rows(p, M)
        trees = np.array([(0, 0, 0, M)], abi.TREE_DT)
        tiles, jobs, parts = host.plan_tiles(trees, abi.PlanGroups(2, p, diff=True), 0, None, host.options_mi355x(p.rows_per_tile, 4))
        passes.append(device.DiffPass(p, device.diff_params(none, None, 0.0, 1.0), trees, tiles, jobs, parts, M, np.arange(7, dtype=np.int32), device="cpu",
                                      pool_blocks=7))
    with pytest.raises(abi.EspError, match="rows_per_tile"):
        passes[0].run(none, none, none)
    p.rows_per_tile = 64
    with pytest.raises(abi.EspError, match="rows_per_tile"):
        passes[1].run(none, none, none)


# ---- a workspace sized for the largest pass serves the smaller ones
@pytest.mark.parametrize("dtype", [abi.ESP_F16, abi.ESP_BF16, abi.ESP_F32])
@pytest.mark.parametrize("vocab", [1, 2048, 50257, 128256, 250000])
def test_logits_workspace_grows_with_the_rows(vocab, dtype):
    p = device.logits_params(vocab, dtype, 1)
    sizes = [abi.attn_lib().esp_logits_workspace_bytes(C.byref(p), n) for n in range(1, 1200)]
    assert sizes[0] > 0 and sizes == sorted(sizes)
    bigger = device.logits_params(vocab + 7, dtype, 1)
    assert all(abi.attn_lib().esp_logits_workspace_bytes(C.byref(bigger), n) >= x for n, x in enumerate(sizes, 1))


@pytest.mark.parametrize("D,rank,n_slices", [(8, 8, 1), (256, 8, 2), (5120, 16, 3), (4096, 64, 3), (2560, 128, 4)])
def test_lowrank_workspace_grows_with_tiles_and_rows(D, rank, n_slices):
    p = device.lowrank_params(D, rank, [(64 * i, 64) for i in range(n_slices)], abi.ESP_BF16, D, 256, 100)
    tiles, slots = (1, 2, 7, 8, 9, 63, 64, 65, 127, 128, 129, 600, 4000), (1, 16, 128, 129, 4096, 65535)
    sizes = {}
    for p.rows_per_tile in (16, 64):
        for t in tiles:
            for n in slots:
                sizes[p.rows_per_tile, t, n] = abi.attn_lib().esp_lowrank_workspace_bytes(C.byref(p), t, n)
    for (r, t, n), x in sizes.items():
        assert x >= 4 * n * rank * n_slices
        assert all(x <= y for (_, t2, n2), y in sizes.items() if t2 >= t and n2 >= n), (r, t, n)


# ---- the adapters' records before they are uploaded
def planned(n=40, rows_per_tile=16):
    p = device.lowrank_params(64, 8, [(0, 64)], abi.ESP_F16, 64, 64, 3)
    p.rows_per_tile = rows_per_tile
    order, tiles = host.plan_lowrank(p, np.arange(n) % 4 - 1)
    return p, order, tiles


@pytest.mark.parametrize("rows_per_tile", [16, 64])
@pytest.mark.parametrize("n", [0, 1, 40, 1000])
def test_lowrank_validate_passes_what_the_planner_made(n, rows_per_tile):
    p, order, tiles = planned(n, rows_per_tile)
    device.validate_lowrank(p, order, tiles, n)
    if len(tiles):
        tiles["count"][0] = 0                                         # a tile without rows does nothing
        device.validate_lowrank(p, order, tiles, n)


@pytest.mark.parametrize("field,value,word", [("adapter", 3, "adapter"), ("adapter", -1, "adapter"), ("count", 17, "rows_per_tile"), ("count", -1, "rows"),
                                              ("first", -1, "slots"), ("first", 25, "slots"), ("first", 2**31 - 1, "slots"), ("first", 1, "twice")])
def test_lowrank_validate_refuses_tiles(field, value, word):
    p, order, tiles = planned()
    tiles[-1][field] = value
    with pytest.raises(abi.EspError, match=word):
        device.validate_lowrank(p, order, tiles, 40)


def test_lowrank_validate_refuses_rows_and_arguments():
    p, order, tiles = planned()
    with pytest.raises(abi.EspError, match="row 39 of 39"):
        device.validate_lowrank(p, order, tiles, 39)
    for row, word in ((-1, "row -1"), (int(order[5]), "twice")):
        bad = order.copy()
        bad[0] = row
        with pytest.raises(abi.EspError, match=word):
            device.validate_lowrank(p, bad, tiles, 40)
    with pytest.raises(abi.EspError, match="twice"):
        device.validate_lowrank(p, order, np.concatenate([tiles, tiles]), 40)
    err = C.create_string_buffer(256)
    for args in ((None, 1, tiles.ctypes.data, 1, 40), (order.ctypes.data, 1, None, 1, 40), (None, -1, None, 0, 40), (None, 0, None, -1, 40), (None, 0, None, 0, -1)):
        assert abi.attn_lib().esp_lowrank_validate(C.byref(p), *args, err, 256) == 1
    p.rows_per_tile = 17
    assert abi.attn_lib().esp_lowrank_validate(C.byref(p), None, 0, None, 0, 40, err, 256) == 2
    assert abi.attn_lib().esp_lowrank_validate(None, None, 0, None, 0, 40, err, 256) == 1


# ---- the logits' arrays that may be NULL
@pytest.mark.parametrize("count,arrays", [("n_slots", ("seen", "counts")), ("n_masks", ("masks",)), ("n_bias", ("bias_tokens", "bias_values"))])
def test_logits_arrays_may_be_null_where_they_are_counted_as_empty(count, arrays):
    """As the header says: by the count in the parameters, not by what the rows in device memory name. The last check of a call, the
    workspace's, is reached where the arrays are accepted."""
    at = {k: 0x1000 for k in ("bias_tokens", "bias_values", "masks", "seen", "counts")}
    err = C.create_string_buffer(256)
    for n, rc in ((0, 4), (2, 1)):
        p = device.logits_params(100, abi.ESP_F16, 2, 2, 2)
        setattr(p, count, n)
        for missing in [(a,) for a in arrays] + [arrays]:
            a = {k: None if k in missing else v for k, v in at.items()}
            assert abi.attn_lib().esp_logits_process(C.byref(p), 0x1000, None, 0x1000, 0x1000, 3, a["bias_tokens"], a["bias_values"], a["masks"], a["seen"],
                                                     a["counts"], 0, None, 0, None, err, 256) == rc, (n, missing, err.value)
