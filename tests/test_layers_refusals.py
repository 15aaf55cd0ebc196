"""What esp_linear_attn and esp_attn_shaped refuse on the host, before anything is launched, their host-side checks and planners. No
GPU: every call here is refused or does nothing."""
import ctypes as C

import numpy as np
import pytest

from espetero_amd import abi, device, host, synth

X = 0x1000                                  # an address that no refused call touches
BIG = 2**31 - 1


def call(fn, *args):
    err = C.create_string_buffer(256)
    rc = getattr(abi.attn_lib(), fn)(*args, err, 256)
    return rc, err.value.decode()


# ---- linear attention
def linear_params(H=8, Hk=4, dk=128, dv=128, n_states=6, row_decay=False, **kw):
    p = device.linear_params(H, Hk, dk, dv, abi.ESP_BF16, dk ** -0.5, n_states, row_decay=row_decay)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def linear_args(p, **kw):
    a = dict(Q=X, K=X, V=X, decay=X, states=X, O=X, tiles=X, n_tiles=2, n_few=1, n_parts=0, n_rows=100, ws=None, nbytes=0)
    a.update(kw)
    return (C.byref(p) if p else None, a["Q"], a["K"], a["V"], a["decay"], a["states"], a["O"], a["tiles"], a["n_tiles"], a["n_few"], a["n_parts"],
            a["n_rows"], a["ws"], a["nbytes"], None)


BAD_LINEAR = [
    (dict(dtype=2), 1, "dtype"), (dict(H=0), 1, "H="), (dict(Hk=0), 1, "H="), (dict(H=9, v_ld=1 << 12, o_ld=1 << 12), 1, "multiple"), (dict(H=-8), 1, "H="),
    (dict(H=4100, v_ld=1 << 20, o_ld=1 << 20), 1, "4096"), (dict(dk=96), 2, "dk"), (dict(dk=256, q_ld=2048, k_ld=2048), 2, "dk"), (dict(dv=96), 2, "dv"),
    (dict(dv=576, v_ld=8192, o_ld=8192), 2, "dv"), (dict(dv=0), 2, "dv"), (dict(q_ld=504), 1, "q_ld"), (dict(k_ld=504), 1, "k_ld"), (dict(v_ld=1016), 1, "v_ld"),
    (dict(o_ld=1016), 1, "o_ld"), (dict(q_ld=516), 1, "multiples"), (dict(o_ld=1028), 1, "multiples"), (dict(v_ld=(1 << 24) + 8), 2, "strides"),
    (dict(decay_ld=7), 1, "decay_ld"), (dict(decay_ld=-1), 1, "decay_ld"), (dict(n_states=-1), 1, "n_states"), (dict(scale=float("nan")), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale")]


@pytest.mark.parametrize("kw,rc,word", BAD_LINEAR)
def test_linear_refuses_parameters(kw, rc, word):
    got = call("esp_linear_attn", *linear_args(linear_params(**kw)))
    assert got[0] == rc and word in got[1], got
    p = linear_params(**kw)
    assert abi.attn_lib().esp_linear_workspace_bytes(C.byref(p), 3) == 0
    n = C.c_int32()
    assert call("esp_linear_hint", C.byref(p), 0, C.byref(n))[0] == rc
    assert call("esp_linear_validate", C.byref(p), None, 0, 0, 0, 0)[0] == rc


@pytest.mark.parametrize("a,rc,word", [
    (dict(Q=None), 1, "Q"), (dict(K=None), 1, "K"), (dict(V=None), 1, "V"), (dict(O=None), 1, "O"), (dict(tiles=None), 1, "tiles"), (dict(decay=None), 1, "decay"),
    (dict(states=None), 1, "states"), (dict(Q=X + 8), 1, "aligned"), (dict(K=X + 2), 1, "aligned"), (dict(V=X + 4), 1, "aligned"), (dict(O=X + 8), 1, "aligned"),
    (dict(states=X + 4), 1, "aligned"), (dict(n_tiles=-1), 1, "counts"), (dict(n_few=3), 1, "counts"), (dict(n_few=-1), 1, "counts"),
    (dict(n_rows=-1), 1, "counts"), (dict(n_parts=-1), 1, "counts"), (dict(n_tiles=70000), 2, "65535"), (dict(n_tiles=70000, n_few=70000), 2, "65535"),
    (dict(n_parts=2), 4, "workspace"), (dict(n_parts=2, ws=X, nbytes=1000), 4, "workspace"), (dict(n_parts=2, ws=X + 8, nbytes=1 << 30), 1, "aligned")])
def test_linear_refuses_arguments(a, rc, word):
    got = call("esp_linear_attn", *linear_args(linear_params(), **a))
    assert got[0] == rc and word in got[1], got


def test_linear_without_tiles_does_nothing():
    assert call("esp_linear_attn", *linear_args(linear_params(), n_tiles=0, n_few=0, tiles=None, Q=None, states=None))[0] == 0
    assert call("esp_linear_attn", *linear_args(None))[0] == 1
    assert "decay" in call("esp_linear_attn", *linear_args(linear_params(), n_rows=0, decay=None))[1]        # the second tile is the chunked kernel's
    assert call("esp_linear_hint", C.byref(linear_params()), 0, None)[0] == 1


@pytest.mark.parametrize("dims", [(64, 64), (128, 192), (128, 512)])
def test_linear_workspace_grows(dims):
    p = linear_params(H=5, Hk=1, dk=dims[0], dv=dims[1])
    sizes = [abi.attn_lib().esp_linear_workspace_bytes(C.byref(p), n) for n in (0, 1, 2, 9, 1000, 1 << 20)]
    assert sizes == sorted(sizes) and all(s >= n * 5 * (dims[0] * dims[1] * 4 + 8) for s, n in zip(sizes, (0, 1, 2, 9, 1000, 1 << 20)))


def seqs(*rows):
    return np.array(list(rows), abi.LINEAR_SEQ_DT)


@pytest.mark.parametrize("workgroups", [1, 2, 64, 512, 5000, BIG])
@pytest.mark.parametrize("rows", [[], [0], [1], [16], [17], [63, 64, 65], [1] * 30 + [700], [5000], [40, 16, 0, 900, 3, 128], [20000, 100], [2048] * 4, [300] * 50])
def test_linear_plans_cover_every_row_once(rows, workgroups):
    p = linear_params(n_states=2 * len(rows))
    base = np.cumsum([7] + rows)[:-1].tolist()
    s = seqs(*[(b, m, i if i % 3 else -1, len(rows) + i if i % 4 else -1) for i, (b, m) in enumerate(zip(base, rows))])
    n_rows = 7 + sum(rows) + 3
    tiles, n_few, n_parts = host.plan_linear(p, s, n_rows, workgroups)
    device.validate_linear(p, tiles, n_few, n_parts, n_rows)
    seen = np.zeros(n_rows, int)
    for t in tiles:
        seen[t["row0"]:t["row0"] + t["rows"]] += 1
    assert (seen[:7] == 0).all() and (seen[7:7 + sum(rows)] == 1).all() and (seen[7 + sum(rows):] == 0).all()
    assert all(t["rows"] <= 16 and t["part"] == -1 for t in tiles[:n_few]) and all(t["rows"] > 0 for t in tiles[n_few:])
    wanted = {(int(q["src"]), int(q["dst"])) for q in s if q["rows"] or q["src"] != q["dst"]}
    assert {(int(t["src"]), int(t["dst"])) for t in tiles if t["after"] == 0} == wanted
    for t in tiles[n_few:]:
        if t["after"]:
            assert t["rows"] % 64 == 0 and t["dst"] == -1
    firsts = [t for t in tiles if t["part"] >= 0 and t["before"] == 0]
    assert sum(int(t["after"]) + 1 for t in firsts) == n_parts


def test_linear_plans_cut_long_sequences_and_leave_full_passes_whole():
    tiles, _, n_parts = host.plan_linear(linear_params(), seqs((0, 16000, 0, 0)), 16000, 512)
    assert len(tiles) > 4 and n_parts == len(tiles)
    whole = seqs(*[(500 * i, 500, i, i) for i in range(256)])
    tiles, _, n_parts = host.plan_linear(linear_params(n_states=256), whole, 128000, 512)
    assert len(tiles) == 256 and n_parts == 0


@pytest.mark.parametrize("rows,word", [
    ([(0, 5, 0, 0), (4, 3, 1, 1)], "row 4"), ([(0, 101, 0, 0)], "outside"), ([(-1, 5, 0, 0)], "outside"), ([(0, -1, 0, 0)], "outside"), ([(BIG, BIG, 0, 0)], "outside"),
    ([(0, 1, 6, 0)], "slots"), ([(0, 1, 0, 6)], "slots"), ([(0, 1, -2, 0)], "slots"), ([(0, 1, 0, -2)], "slots"),
    ([(0, 1, 0, 3), (1, 1, 1, 3)], "slot 3"), ([(0, 1, 0, 1), (1, 1, 1, 2)], "slot 1"), ([(0, 1, 1, 1), (1, 1, 1, -1)], "slot 1"), ([(0, 0, 1, 2), (0, 1, 2, -1)], "slot 2")])
def test_linear_planner_refuses_sequences(rows, word):
    with pytest.raises(abi.EspError, match=word):
        host.plan_linear(linear_params(), seqs(*rows), 100, 512)


def test_linear_planner_refuses_arguments():
    for kw in (dict(workgroups=0), dict(workgroups=-4), dict(n_rows=-1)):
        with pytest.raises(abi.EspError):
            host.plan_linear(linear_params(), seqs((0, 1, 0, 0)), kw.get("n_rows", 10), kw.get("workgroups", 512))
    for kw in (dict(dk=32), dict(dv=100), dict(H=0), dict(n_states=-1)):
        with pytest.raises(abi.EspError):
            host.plan_linear(linear_params(**kw), seqs((0, 1, 0, 0)), 10, 512)
    small, err, n, m, k = np.empty(1, abi.LINEAR_TILE_DT), C.create_string_buffer(256), C.c_int32(), C.c_int32(), C.c_int32()
    s, p = seqs((0, 1, 0, 0), (1, 1, 1, 1), (2, 30, 2, 2)), linear_params()
    assert host.engine_lib().esp_plan_linear(C.byref(p), s.ctypes.data, 3, 40, 512, small.ctypes.data, 1, C.byref(n), C.byref(m), C.byref(k), err, 256) == 4
    assert (n.value, m.value, k.value) == (3, 2, 0)


def planned():
    """Two sequences of few rows, one of 40, one of 1100 in several segments."""
    p = linear_params()
    tiles, n_few, n_parts = host.plan_linear(p, seqs((0, 1, 0, 0), (1, 3, 1, 2), (4, 40, -1, 3), (44, 1100, 4, 4)), 1200, 512)
    assert n_few == 2 and n_parts >= 3
    return p, tiles, n_few, n_parts


@pytest.mark.parametrize("tile,field,value,word", [
    (0, "row0", 1200, "outside"), (0, "row0", -1, "outside"), (0, "rows", -1, "outside"), (0, "rows", BIG, "outside"), (0, "rows", 17, "few"), (0, "row0", 1, "another tile"),
    (2, "row0", 5, "another tile"), (1, "src", 6, "slots"), (1, "src", -2, "slots"), (1, "dst", 6, "slots"), (1, "dst", -2, "slots"), (1, "dst", 0, "another sequence"),
    (0, "dst", 1, "slot 1"), (2, "before", -1, "negative"), (2, "after", -1, "negative"), (2, "part", -2, "negative"), (2, "part", 0, "segments"), (1, "part", 0, "segments"),
    (2, "after", 1, "segments"), (3, "part", 1, "records"), (3, "part", BIG, "records"), (3, "dst", 5, "front"), (4, "before", 0, "record|missing"), (4, "src", 3, "go on"),
    (4, "row0", 60, "another tile"), (-1, "after", 1, "segment|go on|records"), (-1, "before", 1, "go on|segment")])
def test_linear_validate_refuses_tiles(tile, field, value, word):
    p, tiles, n_few, n_parts = planned()
    device.validate_linear(p, tiles, n_few, n_parts, 1200)
    tiles[tile][field] = value
    with pytest.raises(abi.EspError, match=word):
        device.validate_linear(p, tiles, n_few, n_parts, 1200)


def test_linear_validate_refuses_counts_and_missing_segments():
    p, tiles, n_few, n_parts = planned()
    for args in ((tiles, n_few, n_parts - 1, 1200), (tiles, n_few, n_parts, 1143), (tiles, len(tiles) + 1, n_parts, 1200), (tiles, -1, n_parts, 1200),
                 (tiles[:-1], n_few, n_parts, 1200), (np.delete(tiles, 4), n_few, n_parts, 1200), (tiles, len(tiles), n_parts, 1200), (tiles[::-1], 0, n_parts, 1200)):
        with pytest.raises(abi.EspError):
            device.validate_linear(p, *args)
    empty = tiles[:1].copy()
    empty["rows"] = 0                                                  # a tile without rows moves a state
    device.validate_linear(p, empty, 1, 0, 0)


# ---- attention with shaped scores
def shaped_args(p, s, **kw):
    a = dict(Q=X, pool=X, blocks=X, O=X, tiles=X, n_tiles=1, trees=X, n_trees=1, jobs=None, n_jobs=0, n_parts=0, n_rows=1, ws=None, nbytes=0)
    a.update(kw)
    return (C.byref(p) if p else None, C.byref(s) if s else None, a["Q"], a["pool"], a["blocks"], a["O"], a["tiles"], a["n_tiles"], a["trees"], a["n_trees"],
            a["jobs"], a["n_jobs"], a["n_parts"], a["n_rows"], a["ws"], a["nbytes"], None)


def shaped_params(**kw):
    p = synth.make_params(8, 4, 128, abi.ESP_F16, 16, rows_per_tile=1)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


S = abi.ShapeParams(None, None, 0.0, 0)


@pytest.mark.parametrize("p,rc,word", [
    (dict(head_dim=512, q_ld=4096, kv_ld=2048), 2, "head_dim"), (dict(head_dim=64), 2, "head_dim"), (dict(H=7), 1, "multiple"), (dict(dtype=2), 1, "dtype"),
    (dict(bt=24), 1, "bt"), (dict(q_ld=8), 1, "q_ld"), (dict(q_ld=1028), 1, "q_ld"), (dict(kv_base=4), 1, "kv_base"), (dict(gate=X), 2, "gate"),
    (dict(bidi=1), 2, "bidirectional"), (dict(scale=0.0), 1, "scale"), (dict(scale=-1.0), 1, "scale"), (dict(scale=float("nan")), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale"), (dict(scale=1e-30), 1, "scale"), (dict(scale=1e30), 1, "scale"), (dict(window=-1), 1, "window"), (dict(H=258, Hkv=2, q_ld=258 * 128), 2, "128"), (dict(rows_per_tile=0), 2, "rows_per_tile"),
    (dict(rows_per_tile=65), 2, "rows_per_tile"), (dict(rows_per_tile=BIG), 2, "rows_per_tile")])
def test_shaped_refuses_parameters(p, rc, word):
    got = call("esp_attn_shaped", *shaped_args(shaped_params(**p), S))
    assert got[0] == rc and word in got[1], got
    n, g = C.c_int32(), C.c_int32()
    assert call("esp_attn_shaped_hint", C.byref(shaped_params(**p)), 0, C.byref(n), C.byref(g))[0] == rc
    if word != "rows_per_tile":
        assert abi.attn_lib().esp_attn_shaped_rows(C.byref(shaped_params(**p)), 1) == 0
        with pytest.raises(abi.EspError):
            device.attn_shaped_rows(shaped_params(**p), 1)


@pytest.mark.parametrize("a,rc,word", [
    (dict(Q=None), 1, "Q"), (dict(O=None), 1, "O"), (dict(pool=None), 1, "kv_pool"), (dict(tiles=None), 1, "tiles"), (dict(trees=None), 1, "trees"),
    (dict(blocks=None), 1, "blocks"), (dict(n_tiles=-1), 1, "negative"), (dict(n_trees=0), 1, "without"), (dict(n_rows=0), 1, "without"),
    (dict(n_tiles=65536), 2, "65535"), (dict(n_jobs=1, n_parts=2), 1, "jobs"), (dict(n_parts=2), 1, "jobs"), (dict(jobs=X, n_jobs=1), 1, "jobs"),
    (dict(jobs=X, n_jobs=1, n_parts=2), 4, "workspace"), (dict(jobs=X, n_jobs=1, n_parts=2, ws=X, nbytes=100), 4, "workspace"),
    (dict(jobs=X, n_jobs=1, n_parts=2, ws=X + 4, nbytes=1 << 30), 1, "aligned")])
def test_shaped_refuses_arguments(a, rc, word):
    got = call("esp_attn_shaped", *shaped_args(shaped_params(), S, **a))
    assert got[0] == rc and word in got[1], got


def test_shaped_refuses_shapes():
    for cap in (-1.0, float("nan"), float("inf"), float("-inf"), 3e38, 1e-30):
        got = call("esp_attn_shaped", *shaped_args(shaped_params(), abi.ShapeParams(None, None, cap, 0)))
        assert got[0] == 1 and "cap" in got[1], got
    got = call("esp_attn_shaped", *shaped_args(shaped_params(), abi.ShapeParams(None, X + 4, 0.0, 0)))
    assert got[0] == 1 and "spans" in got[1], got
    got = call("esp_attn_shaped", *shaped_args(shaped_params(), abi.ShapeParams(X + 2, None, 0.0, 0)))
    assert got[0] == 1 and "slopes" in got[1], got
    assert call("esp_attn_shaped", *shaped_args(None, S))[0] == 1
    assert call("esp_attn_shaped", *shaped_args(shaped_params(), None))[0] == 1
    assert call("esp_attn_shaped", *shaped_args(shaped_params(), S, n_tiles=0, Q=None))[0] == 0


def test_shaped_rows_and_workspace():
    lib = abi.attn_lib()
    for H, Hkv, hd in ((8, 4, 128), (16, 4, 256), (10, 2, 128), (128, 1, 256), (40, 40, 128)):
        p = shaped_params(H=H, Hkv=Hkv, head_dim=hd, q_ld=H * hd, kv_ld=Hkv * hd)
        for rows in (1, 2, 3, 4, 5, 8, 16, 17, 100, 3000, BIG):
            p.rows_per_tile = r = lib.esp_attn_shaped_rows(C.byref(p), rows)
            assert 1 <= r <= min(rows, 128 * Hkv // H), (H, Hkv, rows)
            sizes = [lib.esp_attn_shaped_workspace_bytes(C.byref(p), n) for n in (0, 1, 3, 1000)]
            assert sizes == sorted(sizes) and sizes[2] >= 3 * r * H * (hd + 2) * 4
    assert lib.esp_attn_shaped_rows(C.byref(shaped_params()), 0) == 0


def test_shaped_validates_records():
    p = shaped_params()
    trees = np.array([(0, 40, 0, 1)], abi.TREE_DT)
    blocks = np.arange(3, dtype=np.int32)
    tile = (0, 0, 0, 40, -1, 1, 0, 1)
    ok = lambda t=tile, tr=trees, b=blocks, pool=3, q=p: device.validate(q, np.array([t], abi.TILE_DT), tr, np.zeros(0, abi.COMBINE_DT), 0, 1, b, pool,  # noqa: E731
                                                                         shaped=True)
    ok()
    ok((0, 0, 16, BIG, -1, 1, 0, 1))
    with pytest.raises(abi.EspError, match="do not meet"):
        ok((0, 0, 0, 32, -1, 1, 0, 1))
    with pytest.raises(abi.EspError, match="block"):
        ok(tr=np.array([(0, 48, 0, 1)], abi.TREE_DT), t=(0, 0, 0, 48, -1, 1, 0, 1))      # the row's own key has no block
    with pytest.raises(abi.EspError, match="block"):
        ok(pool=2)
    with pytest.raises(abi.EspError, match="ring"):
        ok(q=shaped_params(window=40, ring=1), pool=1, t=(0, 0, 1, 40, -1, 1, 0, 1))
    with pytest.raises(abi.EspError, match="rows_per_tile"):
        ok(q=shaped_params(rows_per_tile=65))
    with pytest.raises(abi.EspError, match="gate"):
        ok(q=shaped_params(gate=X))
    for other in (dict(diff=True), dict(rows_in_pool=True)):
        with pytest.raises(abi.EspError, match="mode"):
            device.validate(p, np.array([tile], abi.TILE_DT), trees, np.zeros(0, abi.COMBINE_DT), 0, 1, blocks, 3, shaped=True, **other)


@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("heads", [(8, 4, 128), (32, 4, 256), (64, 1, 128), (128, 1, 256)])
@pytest.mark.parametrize("pairs", [[(0, 1)], [(900, 1), (5000, 1), (17, 1)], [(3000, 5)] * 3, [(0, 700), (40, 33), (2000, 129)], [(12000, 500)], [(0, 1), (30000, 64)]])
def test_shaped_plans_cover_every_key_once(pairs, heads, window):
    p = synth.make_params(*heads, abi.ESP_F16, 16, window=window, rows_per_tile=1)
    p.rows_per_tile = device.attn_shaped_rows(p, max(M for _, M in pairs))
    trees, at, used = np.zeros(len(pairs), abi.TREE_DT), 0, 0
    for i, (P, M) in enumerate(pairs):
        trees[i] = (at, P, used, M)
        at, used = at + M, used + -(-(P + M) // 16)
    pos = np.zeros((at, 4), np.int32)
    for b, P, _, M in trees:
        pos[b:b + M, :3] = (P + np.arange(M))[:, None]
    for resident in (64, 256, 4096):
        tiles, jobs, n_parts = host.plan_tiles(trees, abi.PlanGroups(heads[1], p, shaped=True), window, pos if window else None,
                                               host.options_mi355x(p.rows_per_tile, resident))
        device.validate(p, tiles, trees, jobs, n_parts, at, np.arange(used, dtype=np.int32), used, shaped=True)
        rows = set()
        for tree in range(len(pairs)):
            base, P, _, M = (int(x) for x in trees[tree])
            mine = tiles[tiles["tree"] == tree]
            for r0 in sorted({int(r) for r in mine["r0"]}):
                n = min(p.rows_per_tile, base + M - r0)
                rows |= set(range(r0, r0 + n))
                first = P + r0 - base
                spans = []
                for x in mine[mine["r0"] == r0]:
                    lo, hi = int(x["k0"]), min(int(x["k1"]), P)
                    if x["last"]:
                        lo = P + int(x["b0"]) if hi <= lo else lo
                        hi = P + int(x["last"]) - 1 if x["last"] >= 2 else P + M
                    spans.append((lo, max(lo, hi)))
                spans.sort()
                assert spans[0][0] <= (max(0, first - window + 1) if window else 0) and spans[-1][1] == P + M      # a prefix may end at the last row
                assert all(x[1] == y[0] for x, y in zip(spans, spans[1:]))
        assert rows == set(range(at))
        parts = tiles["part"][tiles["part"] >= 0]
        assert len(set(parts)) == len(parts) == n_parts == jobs["nparts"].sum()


@pytest.mark.parametrize("heads", [(32, 1, 256), (128, 1, 128)])
@pytest.mark.parametrize("P", [0, 1, 15, 16, 31, 32, 64, 96, 128, 500, 512, 4096, 16000])
def test_shaped_plans_grow_with_a_chain(P, heads):
    """Single tokens on the tiled kernel: open-ended tiles cover every key once, however far the chain has moved on."""
    p = synth.make_params(*heads, abi.ESP_F16, 16, rows_per_tile=1)
    trees = np.array([(0, P, 0, 1), (1, P // 2, P // 16 + 4, 1)], abi.TREE_DT)
    for resident in (8, 256, 5000):
        tiles, jobs, n_parts = host.plan_tiles(trees, abi.PlanGroups(1, p, shaped=True), 0, None, host.options_mi355x(1, resident))
        tiles = host.open_ended(tiles, trees)
        assert P < 4096 or resident < 256 or n_parts > 2
        for s in (0, 1, 2, 15, 16, 17, 100):
            for i, t in enumerate(trees):
                now, spans = int(t["P"]) + s, []
                for x in tiles[tiles["tree"] == i]:                           # what the kernel makes of a record
                    k1 = min(int(x["k1"]), now)
                    lo = now + int(x["b0"]) if x["last"] and k1 <= x["k0"] else int(x["k0"])
                    hi = k1 if not x["last"] else now + int(x["last"]) - 1 if x["last"] >= 2 else now + 1
                    spans.append((lo, min(hi, now + 1)))
                spans.sort()
                assert spans[0][0] == 0 and spans[-1][1] == now + 1 and all(a[1] == b[0] for a, b in zip(spans, spans[1:])), (s, spans)


def test_shaped_pass_refuses_spans_of_another_shape():
    p = shaped_params()
    trees, tiles = np.array([(0, 40, 0, 1)], abi.TREE_DT), np.array([(0, 0, 0, 40, -1, 1, 0, 1)], abi.TILE_DT)
    for spans in (np.zeros((2, 2), np.int32), np.zeros(2, np.int32), np.zeros((1, 3), np.int32)):
        with pytest.raises(abi.EspError, match="spans"):
            device.ShapedPass(p, device.shape_params(), trees, tiles, np.zeros(0, abi.COMBINE_DT), 0, 1, np.arange(3, dtype=np.int32), spans=spans, device="cpu")


def test_calls_refuse_other_records():
    from espetero_amd import _calls
    lp, sp, ap = linear_params(), device.shape_params(), shaped_params()
    with pytest.raises(TypeError):
        _calls.linear_attn(ap, *[None] * 7, 0, 0, 0, 0, None, 0, 0)
    with pytest.raises(TypeError):
        _calls.attn_shaped(ap, lp, *[None] * 5, 0, None, 0, None, 0, 0, 0, None, 0, 0)
    with pytest.raises(TypeError):
        _calls.attn_shaped(lp, sp, *[None] * 5, 0, None, 0, None, 0, 0, 0, None, 0, 0)
    _calls.linear_attn(lp, *[None] * 7, 0, 0, 0, 0, None, 0, 0)                                # no tiles: nothing to do
    _calls.attn_shaped(ap, sp, *[None] * 5, 0, None, 0, None, 0, 0, 0, None, 0, 0)
