"""What esp_attn_diff, esp_lowrank_add and esp_logits_process refuse on the host, before anything is launched, their host-side
checks and planners. No GPU: every call here is refused or does nothing."""
import ctypes as C

import numpy as np
import pytest

from espetero_amd import abi, device, host, synth

X = 0x1000                                  # an address that no refused call touches


def call(fn, *args):
    err = C.create_string_buffer(256)
    rc = getattr(abi.attn_lib(), fn)(*args, err, 256)
    return rc, err.value.decode()


# ---- differential attention
def diff_args(p, d, **kw):
    a = dict(Q=X, pool=X, blocks=X, O=X, tiles=X, n_tiles=1, trees=X, n_trees=1, jobs=None, n_jobs=0, n_parts=0, n_rows=1, ws=None, nbytes=0)
    a.update(kw)
    return (C.byref(p) if p else None, C.byref(d) if d else None, a["Q"], a["pool"], a["blocks"], a["O"], a["tiles"], a["n_tiles"], a["trees"], a["n_trees"],
            a["jobs"], a["n_jobs"], a["n_parts"], a["n_rows"], a["ws"], a["nbytes"], None)


def diff_params(**kw):
    p = synth.make_params(8, 4, 128, abi.ESP_F16, 16, rows_per_tile=1)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


D = abi.DiffParams(X, X, 1e-5, 1.0)


@pytest.mark.parametrize("p,rc,word", [
    (dict(head_dim=256, q_ld=2048, kv_ld=1024), 2, "head_dim"), (dict(head_dim=512, q_ld=4096, kv_ld=2048), 2, "head_dim"), (dict(head_dim=64), 2, "head_dim"),
    (dict(H=6, Hkv=3), 1, "pairs"), (dict(H=7), 1, "multiple"), (dict(dtype=2), 1, "dtype"), (dict(bt=24), 1, "bt"), (dict(q_ld=8), 1, "q_ld"),
    (dict(q_ld=1028), 1, "q_ld"), (dict(kv_base=4), 1, "kv_base"), (dict(gate=X), 2, "gate"), (dict(bidi=1), 2, "bidi"), (dict(scale=0.0), 1, "scale"),
    (dict(scale=float("nan")), 1, "scale"), (dict(window=-1), 1, "window"), (dict(rows_per_tile=0), 2, "rows_per_tile"),
    (dict(rows_per_tile=1 << 20), 2, "rows_per_tile")])
def test_diff_refuses_parameters(p, rc, word):
    got = call("esp_attn_diff", *diff_args(diff_params(**p), D))
    assert got[0] == rc and word in got[1], got
    if word != "rows_per_tile":
        assert abi.attn_lib().esp_attn_diff_rows(C.byref(diff_params(**p)), 1) == 0


@pytest.mark.parametrize("a,rc,word", [
    (dict(Q=None), 1, "Q"), (dict(O=None), 1, "O"), (dict(pool=None), 1, "kv_pool"), (dict(tiles=None), 1, "tiles"), (dict(trees=None), 1, "trees"),
    (dict(blocks=None), 1, "blocks"), (dict(n_tiles=-1), 1, "negative"), (dict(n_trees=0), 1, "without"), (dict(n_rows=0), 1, "without"),
    (dict(n_tiles=65536), 2, "65535"), (dict(n_jobs=1, n_parts=2), 1, "jobs"), (dict(n_parts=2), 1, "jobs"), (dict(jobs=X, n_jobs=1), 1, "jobs"),
    (dict(jobs=X, n_jobs=1, n_parts=2), 4, "workspace"), (dict(jobs=X, n_jobs=1, n_parts=2, ws=X, nbytes=100), 4, "workspace"),
    (dict(jobs=X, n_jobs=1, n_parts=2, ws=X + 4, nbytes=1 << 30), 1, "aligned")])
def test_diff_refuses_arguments(a, rc, word):
    got = call("esp_attn_diff", *diff_args(diff_params(), D, **a))
    assert got[0] == rc and word in got[1], got


def test_diff_refuses_records_that_are_missing():
    assert call("esp_attn_diff", *diff_args(None, D))[0] == 1
    assert call("esp_attn_diff", *diff_args(diff_params(), None))[0] == 1
    assert call("esp_attn_diff", *diff_args(diff_params(), abi.DiffParams(None, X, 1e-5, 1.0)))[0] == 1
    assert call("esp_attn_diff", *diff_args(diff_params(), abi.DiffParams(X, X, -1.0, 1.0)))[0] == 1
    assert call("esp_attn_diff", *diff_args(diff_params(), D, n_tiles=0, Q=None))[0] == 0


def test_diff_rows_and_workspace():
    lib = abi.attn_lib()
    for H, Hkv in ((8, 4), (16, 4), (10, 2), (32, 2)):
        p = diff_params(H=H, Hkv=Hkv, q_ld=H * 128, kv_ld=Hkv * 128)
        for rows in (1, 2, 3, 4, 5, 8, 16, 17, 100, 3000):
            r = lib.esp_attn_diff_rows(C.byref(p), rows)
            assert 1 <= r, (H, Hkv, rows)
            p.rows_per_tile = r
            err, n, g = C.create_string_buffer(256), C.c_int32(), C.c_int32()
            need = lib.esp_attn_diff_workspace_bytes(C.byref(p), 3)
            assert need >= 3 * r * H * (256 + 2) * 4                    # both maps' records
    assert lib.esp_attn_diff_rows(C.byref(diff_params()), 0) == 0


def test_diff_validates_records():
    p = diff_params()
    trees = np.array([(0, 40, 0, 1)], abi.TREE_DT)
    blocks = np.arange(3, dtype=np.int32)
    tile = (0, 0, 0, 40, -1, 1, 0, 1)
    ok = lambda t=tile, tr=trees, b=blocks, pool=3, q=p: device.validate(q, np.array([t], abi.TILE_DT), tr, np.zeros(0, abi.COMBINE_DT), 0, 1, b, pool,  # noqa: E731
                                                                         diff=True)
    ok()
    ok((0, 0, 16, 2**31 - 1, -1, 1, 0, 1))
    with pytest.raises(abi.EspError, match="do not meet"):
        ok((0, 0, 0, 32, -1, 1, 0, 1))
    with pytest.raises(abi.EspError, match="block"):
        ok(tr=np.array([(0, 48, 0, 1)], abi.TREE_DT), t=(0, 0, 0, 48, -1, 1, 0, 1))      # the row's own key has no block
    with pytest.raises(abi.EspError, match="block"):
        ok(pool=2)
    with pytest.raises(abi.EspError, match="ring"):
        ok(q=diff_params(window=40, ring=1), pool=1, t=(0, 0, 1, 40, -1, 1, 0, 1))
    with pytest.raises(abi.EspError, match="pairs"):
        ok(q=diff_params(H=3, Hkv=3))
    with pytest.raises(abi.EspError, match="mode"):
        device.validate(p, np.array([tile], abi.TILE_DT), trees, np.zeros(0, abi.COMBINE_DT), 0, 1, blocks, 3, diff=True, rows_in_pool=True)


# ---- low-rank adapters
def lowrank_params(**kw):
    p = device.lowrank_params(64, 8, [(0, 64), (64, 32)], abi.ESP_F16, 64, 96, 3)
    p.rows_per_tile = abi.attn_lib().esp_lowrank_rows(C.byref(p), 4)
    for k, v in kw.items():
        if k in ("y_off", "width"):
            for i, x in enumerate(v):
                getattr(p, k)[i] = x
        else:
            setattr(p, k, v)
    return p


def lowrank_args(p, **kw):
    a = dict(X=X, A=X, B=X, scale=X, Y=X, order=X, n_slots=4, tiles=X, n_tiles=1, ws=X, nbytes=1 << 30)
    a.update(kw)
    return (C.byref(p) if p else None, a["X"], a["A"], a["B"], a["scale"], a["Y"], a["order"], a["n_slots"], a["tiles"], a["n_tiles"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("p", [dict(dtype=2), dict(D=0), dict(D=12), dict(rank=0), dict(rank=12), dict(rank=136), dict(n_slices=0), dict(n_slices=5),
                               dict(n_adapters=0), dict(x_ld=56), dict(x_ld=68), dict(y_ld=95), dict(width=[64, 0]), dict(y_off=[-1, 64]),
                               dict(y_off=[0, 63]), dict(y_off=[2**31 - 10, 64])])
def test_lowrank_refuses_parameters(p):
    q = lowrank_params(**p)
    assert call("esp_lowrank_add", *lowrank_args(q))[0] == 1
    assert abi.attn_lib().esp_lowrank_rows(C.byref(q), 4) == 0 and abi.attn_lib().esp_lowrank_workspace_bytes(C.byref(q), 1, 4) == 0


@pytest.mark.parametrize("a,rc", [(dict(X=None), 1), (dict(A=None), 1), (dict(B=None), 1), (dict(scale=None), 1), (dict(Y=None), 1), (dict(order=None), 1),
                                  (dict(tiles=None), 1), (dict(n_slots=0), 1), (dict(n_slots=-1), 1), (dict(n_tiles=-1), 1), (dict(ws=None), 4),
                                  (dict(nbytes=10), 4), (dict(X=X + 8), 1), (dict(A=X + 2), 1), (dict(B=X + 4), 1), (dict(ws=X + 4), 1)])
def test_lowrank_refuses_arguments(a, rc):
    assert call("esp_lowrank_add", *lowrank_args(lowrank_params(), **a))[0] == rc
    assert call("esp_lowrank_add", *lowrank_args(lowrank_params(rows_per_tile=7)))[0] == 2
    assert call("esp_lowrank_add", *lowrank_args(None))[0] == 1
    assert call("esp_lowrank_add", *lowrank_args(lowrank_params(), n_tiles=0, X=None))[0] == 0


@pytest.mark.parametrize("n_adapters", [7, 5000, 2**31 - 1])
@pytest.mark.parametrize("rows_per_tile", [1, 16, 2**31 - 1])
def test_lowrank_plans_of_any_table_and_tile(n_adapters, rows_per_tile):
    a = np.random.default_rng(1).integers(-1, min(n_adapters, 40), 300).astype(np.int32)
    a[::50] = n_adapters - 1
    order, tiles = host.plan_lowrank(lowrank_params(n_adapters=n_adapters, rows_per_tile=rows_per_tile), a)
    assert (order == sorted(np.flatnonzero(a >= 0), key=lambda r: (a[r], r))).all()
    assert (tiles["first"] == np.cumsum(tiles["count"]) - tiles["count"]).all() and tiles["count"].sum() == len(order)
    for t in tiles:
        assert 0 < t["count"] <= rows_per_tile and (a[order[t["first"]:t["first"] + t["count"]]] == t["adapter"]).all()
    for x, y in zip(tiles, tiles[1:]):
        assert x["adapter"] < y["adapter"] or (x["adapter"] == y["adapter"] and x["count"] == rows_per_tile)


def test_lowrank_refuses_more_workgroups_than_a_launch_has():
    p = lowrank_params(y_ld=1 << 22)
    p.y_off[0], p.width[0], p.y_off[1], p.width[1] = 0, 1 << 21, 1 << 21, 64
    rc, msg = call("esp_lowrank_add", *lowrank_args(p, n_tiles=65535, n_slots=65535, nbytes=1 << 40))
    assert rc == 2 and "workgroups" in msg, msg
    assert call("esp_lowrank_add", *lowrank_args(p, n_tiles=65536))[0] == 2


def test_lowrank_plan():
    p = lowrank_params(rows_per_tile=2)
    order, tiles = host.plan_lowrank(p, [1, 0, -1, 1, 1, 2, -1, 0])
    assert list(order) == [1, 7, 0, 3, 4, 5]
    assert [tuple(t)[:3] for t in tiles] == [(0, 0, 2), (1, 2, 2), (1, 4, 1), (2, 5, 1)]
    assert all(len(x) == 0 for x in host.plan_lowrank(p, [-1, -1])) and all(len(x) == 0 for x in host.plan_lowrank(p, []))
    for bad in ([0, 3], [0, -2]):
        with pytest.raises(abi.EspError, match="row 1: adapter"):
            host.plan_lowrank(p, bad)
    rng = np.random.default_rng(0)
    a = rng.integers(-1, 3, 1000)
    p.rows_per_tile = 16
    order, tiles = host.plan_lowrank(p, a)
    assert sorted(order) == list(np.flatnonzero(a >= 0)) and tiles["count"].sum() == len(order) and tiles["count"].max() == 16
    for t in tiles:
        assert (a[order[t["first"]:t["first"] + t["count"]]] == t["adapter"]).all()
    small = np.empty(1, abi.LOWRANK_TILE_DT)
    err, n, m, o = C.create_string_buffer(256), C.c_int32(), C.c_int32(), np.empty(1000, np.int32)
    a32 = a.astype(np.int32)
    assert host.engine_lib().esp_plan_lowrank(C.byref(p), a32.ctypes.data, 1000, o.ctypes.data, C.byref(n), small.ctypes.data, 1, C.byref(m), err, 256) == 4
    assert m.value == len(tiles)


@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("heads", [(8, 4), (32, 4), (64, 2)])
@pytest.mark.parametrize("seqs", [[(0, 1)], [(900, 1), (5000, 1), (17, 1)], [(3000, 5)] * 3, [(0, 700), (40, 33), (2000, 129)], [(12000, 500)], [(0, 1), (30000, 64)]])
def test_diff_plans_cover_every_key_once(seqs, heads, window):
    p = synth.make_params(*heads, 128, abi.ESP_F16, 16, window=window, rows_per_tile=1)
    p.rows_per_tile = device.attn_diff_rows(p, max(M for _, M in seqs))
    trees, at, used = np.zeros(len(seqs), abi.TREE_DT), 0, 0
    for i, (P, M) in enumerate(seqs):
        trees[i] = (at, P, used, M)
        at, used = at + M, used + -(-(P + M) // 16)
    pos = np.zeros((at, 4), np.int32)
    for b, P, _, M in trees:
        pos[b:b + M, :3] = (P + np.arange(M))[:, None]
    for resident in (64, 256, 4096):
        tiles, jobs, n_parts = host.plan_tiles(trees, abi.PlanGroups(heads[1] // 2, p, diff=True), window, pos if window else None,
                                               host.options_mi355x(p.rows_per_tile, resident))
        device.validate(p, tiles, trees, jobs, n_parts, at, np.arange(used, dtype=np.int32), used, diff=True)
        rows, length, order = set(), {}, []
        for tree in range(len(seqs)):
            base, P, _, M = trees[tree]
            mine = tiles[tiles["tree"] == tree]
            for r0 in set(mine["r0"]):
                n = min(p.rows_per_tile, base + M - r0)
                rows |= set(range(r0, r0 + n))
                first, end = P + r0 - base, P + r0 - base + n              # the tile's rows see keys up to their own, [.., end) of them
                spans = []
                for x in mine[mine["r0"] == r0]:                             # a part's keys: cached ones, and rows of the pass behind them
                    lo, hi = int(x["k0"]), min(int(x["k1"]), P)
                    if x["last"]:
                        lo = P + int(x["b0"]) if hi <= lo else lo
                        hi = min(end, P + int(x["last"]) - 1) if x["last"] >= 2 else end
                    spans.append((lo, max(lo, hi)))
                spans.sort()
                assert spans[0][0] <= (max(0, first - window + 1) if window else 0) and spans[-1][1] == end
                assert all(x[1] == y[0] for x, y in zip(spans, spans[1:]))
                length[(tree, int(r0))] = sum(y - x for x, y in spans) // len(spans)
        assert rows == set(range(at))
        parts = tiles["part"][tiles["part"] >= 0]
        assert len(set(parts)) == len(parts) == n_parts == jobs["nparts"].sum()
        if p.rows_per_tile * heads[0] // heads[1] > 16 and not window:             # many packed rows: dispatched from the end, the longest parts first
            for x in tiles:
                key = (int(x["tree"]), int(x["r0"]))
                order += [] if key in order else [key]
            assert all(length[y] >= length[x] - 1 for x, y in zip(order, order[1:]))


# ---- logits
def logits_args(p, **kw):
    a = dict(L=X, out=X + 64, tokens=X, rows=X, n=2, bt=X, bv=X, masks=X, seen=X, counts=X, record=0, ws=X, nbytes=1 << 20)
    a.update(kw)
    return (C.byref(p) if p else None, a["L"], a["out"], a["tokens"], a["rows"], a["n"], a["bt"], a["bv"], a["masks"], a["seen"], a["counts"], a["record"],
            a["ws"], a["nbytes"], None)


def logits_params(**kw):
    p = device.logits_params(100, abi.ESP_F16, 3, 2, 5)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("p", [dict(dtype=3), dict(vocab=0), dict(vocab=2**31 - 1), dict(n_slots=-1), dict(n_masks=-1), dict(n_bias=-1), dict(n_bias=2**31 - 1), dict(in_ld=99),
                               dict(out_ld=99)])
def test_logits_refuses_parameters(p):
    assert call("esp_logits_process", *logits_args(logits_params(**p)))[0] == 1


@pytest.mark.parametrize("a,rc", [(dict(L=None), 1), (dict(rows=None), 1), (dict(out=None, tokens=None), 1), (dict(n=-1), 1), (dict(n=65536), 1), (dict(seen=None), 1),
                                  (dict(counts=None), 1), (dict(masks=None), 1), (dict(bt=None), 1), (dict(bv=None), 1), (dict(record=2), 1),
                                  (dict(record=1, tokens=None), 1), (dict(ws=None), 4), (dict(nbytes=4), 4), (dict(ws=X + 2), 1), (dict(out=X), 1)])
def test_logits_refuses_arguments(a, rc):
    assert call("esp_logits_process", *logits_args(logits_params(), **a))[0] == rc
    assert call("esp_logits_process", *logits_args(None))[0] == 1
    assert call("esp_logits_process", *logits_args(logits_params(), n=0, L=None))[0] == 0
    assert call("esp_logits_process", *logits_args(logits_params(n_slots=0), record=1))[0] == 1


def test_histories_refuse():
    p = logits_params()
    for kw in ((X, X, X, X, -1, 0), (None, X, X, X, 1, 0), (X, None, X, X, 1, 0), (X, X, None, X, 1, 0), (X, X, X, None, 1, 0), (X, X, X, X, 1, 2),
               (X, X, X, X, 2**31 - 1, 1)):
        assert call("esp_history_record", C.byref(p), *kw, None)[0] == 1
    assert call("esp_history_record", C.byref(p), None, None, None, None, 0, 1, None)[0] == 0
    for kw in ((X, X, X, -1), (None, X, X, 1), (X, None, X, 1), (X, X, None, 1), (X, X, X, 65536)):
        assert call("esp_history_clear", C.byref(p), *kw, None)[0] == 1
    assert call("esp_history_clear", C.byref(p), None, None, None, 0, None)[0] == 0


@pytest.mark.parametrize("field,value", [("slot", 3), ("slot", -2), ("mask", 2), ("mask", -2), ("repetition", 0.0), ("repetition", float("nan")),
                                         ("frequency", float("inf")), ("presence", float("nan")), ("n_bias", -1), ("n_bias", 6), ("bias0", -1), ("bias0", 3)])
def test_logits_validate(field, value):
    p = logits_params()
    rows = np.zeros(2, abi.LOGITS_ROW_DT)
    rows["repetition"], rows["n_bias"] = 1.0, 3
    tokens = np.array([4, 9, 99, 0, 1], np.int32)
    ok = lambda r, t: call("esp_logits_validate", C.byref(p), r.ctypes.data, len(r), t.ctypes.data)[0]  # noqa: E731
    assert ok(rows, tokens) == 0
    for bad in ([4, 4, 99, 0, 1], [9, 4, 99, 0, 1], [4, 9, 100, 0, 1], [-1, 9, 99, 0, 1]):
        assert ok(rows, np.array(bad, np.int32)) == 1
    rows[1][field] = value
    assert ok(rows, tokens) == 1
