"""Plans of differential attention and of attention with shaped scores on layers with a window: their kernels see a row at its place in the
cache, wherever its rotary position lies."""
import numpy as np
import pytest

from espetero_amd import abi, host, synth


def scanned(tiles, trees):
    """[first, end) of the keys that the tiles of each (tree, first row) scan, in order of their first key."""
    out = {}
    for t in tiles:
        base, P, _, M = (int(x) for x in trees[t["tree"]])
        lo, end = int(t["k0"]), min(int(t["k1"]), P)
        if t["last"]:
            lo = P + int(t["b0"]) if end <= lo else lo
            end = P + (int(t["last"]) - 1 if t["last"] >= 2 else M)
        if end > lo:
            out.setdefault((int(t["tree"]), int(t["r0"]) - base), []).append((lo, end))
    return {k: sorted(v) for k, v in out.items()}


@pytest.mark.parametrize("ahead", [-300, -1, 0, 1, 64, 5000])
@pytest.mark.parametrize("workgroups", [16, 512, 4096])
@pytest.mark.parametrize("kind,heads,hd", [("shaped", (8, 2), 128), ("shaped", (4, 4), 256), ("diff", (8, 4), 128)])
@pytest.mark.parametrize("rows", [1, 3, 90])
@pytest.mark.parametrize("window", [1, 100, 333])
def test_a_window_starts_at_the_rows_place_in_the_cache(window, rows, kind, heads, hd, workgroups, ahead):
    trees, n = np.zeros(3, abi.TREE_DT), 0
    for i, (P, M) in enumerate([(400, rows), (0, rows), (2000, max(1, rows // 2))]):
        trees[i] = (n, P, 200 * i, M)
        n += M
    pos = np.zeros((n, 4), np.int32)
    for base, P, _, M in trees.tolist():
        pos[base:base + M, :3] = (P + ahead + np.arange(M))[:, None]
    p = synth.make_params(*heads, hd, abi.ESP_BF16, 16, window=window, scale=0.1, rows_per_tile=1)
    p.rows_per_tile = R = min(rows, (128 if kind == "shaped" else 64) // (heads[0] // heads[1]))
    groups = abi.PlanGroups(heads[1], p, **{kind: True})
    o = host.options_mi355x(R, workgroups)
    plan = host.plan_tiles(trees, groups, window, pos, o)
    got = scanned(plan[0], trees)
    for i, (base, P, _, M) in enumerate(trees.tolist()):
        for r in range(0, M, R):
            parts = got[i, r]
            assert parts[0][0] <= max(0, P + r - window + 1)
            assert all(x[1] >= y[0] for x, y in zip(parts, parts[1:]))
            assert parts[-1][1] >= P + min(M, r + R)
    for again in (host.plan_tiles(trees, groups, window, None, o),):
        assert all((np.asarray(x) == np.asarray(y)).all() for x, y in zip(plan, again))


def test_a_plain_plan_with_a_window_needs_positions():
    trees = np.array([(0, 400, 0, 2)], abi.TREE_DT)
    with pytest.raises(abi.EspError, match="pos"):
        host.plan_tiles(trees, 4, 100, None, host.options_mi355x(2, 256))
