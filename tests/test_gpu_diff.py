"""esp_attn_diff on the device against the operator in float64."""
import ctypes as C

import numpy as np
import pytest
import torch

from diff_utils import HD, DiffCase
from espetero_amd import abi, device, host
from oracle import binding as ob

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a).view(np.int16 if a.dtype == np.uint16 else a.dtype)).cuda()


class Run:
    def __init__(self, case, rows_per_tile=None, workgroups=None, cut_batch=False, open_ended=False):
        device.init(0)
        self.case, self.p = case, case.params(rows_per_tile)
        self.tiles, self.jobs, self.parts = case.plan(self.p, workgroups, cut_batch)
        tiles = host.open_ended(self.tiles, case.trees) if open_ended else self.tiles
        self.d = device.diff_params(dev(case.weight), dev(case.norm_w), case.eps, case.factor)
        self.dp = device.DiffPass(self.p, self.d, case.trees, tiles, self.jobs, self.parts, case.n_rows, case.block_list, pool_blocks=case.n_blocks)
        self.Q, self.pool = dev(case.Q), dev(case.pool)
        self.O = torch.full((case.n_rows, case.q_ld), 0x1234, dtype=torch.int16, device="cuda")
        print(f"diff H{case.H}/{case.Hkv} bt{case.bt} seqs{case.seqs[:6]} window{case.window} ring{case.ring} rows{self.p.rows_per_tile} "
              f"tiles{len(tiles)} parts{self.parts}", flush=True)

    def __call__(self):
        self.dp.run(self.Q, self.pool, self.O)
        torch.cuda.synchronize()
        return self.bits()

    def bits(self):
        return self.O.cpu().numpy().view(np.uint16).copy()


def check(case, bits, rows=None):
    want, tol = case.expected(rows)
    H = case.H
    got = ob.to_f32(bits, case.dtype).astype(np.float64)
    live = np.isfinite(want[:, 0]) if rows is None else np.array(sorted(rows))
    worst = np.max(np.abs(got[live, :H * HD] - want[live]) / tol[live])
    print(f"  of the bound: {worst:.3f}", flush=True)
    assert np.all(np.abs(got[live, :H * HD] - want[live]) <= tol[live]), worst
    assert (bits[:, H * HD:] == 0x1234).all()                       # columns behind the heads are left as they were


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", [(4, 2), (8, 4), (16, 4), (10, 2), (16, 2), (32, 2), (64, 2), (256, 2)])
@pytest.mark.parametrize("bt,seqs", [(16, [(0, 1), (1, 1), (15, 1), (16, 1), (130, 1), (700, 1)]), (64, [(63, 1), (64, 1), (250, 1)])])
def test_single_tokens(heads, dtype, bt, seqs):
    c = DiffCase(*heads, dtype, bt, seqs, seed=heads[0])
    check(c, Run(c)())
    check(c, Run(c, workgroups=4096)())                              # cut as finely as the planner will


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,rows", [((8, 4), 5), ((16, 4), 4), ((12, 4), 5), ((16, 8), 8), ((4, 4), 16)])
def test_drafts(heads, rows, dtype):
    c = DiffCase(*heads, dtype, 16, [(0, rows), (30, rows - 1), (200, rows), (33, 1)], seed=rows)
    check(c, Run(c)())
    check(c, Run(c, workgroups=4096)())
    check(c, Run(c, rows_per_tile=1)())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,seqs", [((4, 2), [(0, 300)]), ((8, 2), [(50, 133), (0, 17), (7, 64)]), ((8, 4), [(129, 130)]),
                                        ((4, 4), [(0, 129), (31, 127)]), ((10, 2), [(13, 60)]), ((64, 2), [(40, 9), (0, 3)])])
def test_prompts_and_chunks(heads, seqs, dtype):
    c = DiffCase(*heads, dtype, 16, seqs, seed=3)
    check(c, Run(c)())
    check(c, Run(c, workgroups=2048, cut_batch=True)())


@pytest.mark.parametrize("ring", [False, True])
@pytest.mark.parametrize("window", [1, 16, 100])
@pytest.mark.parametrize("seqs", [[(0, 1), (99, 1), (100, 1), (431, 1)], [(0, 3), (200, 4)], [(0, 90), (150, 140)]])
def test_windows(seqs, window, ring):
    c = DiffCase(8, 4, F16, 16, seqs, window=window, ring=ring, seed=window)
    check(c, Run(c)())
    check(c, Run(c, workgroups=2048)())


def test_sharp_softmax_and_no_norm():
    for norm in (True, False):
        c = DiffCase(8, 2, F16, 16, [(500, 1), (90, 3), (60, 70)], seed=5, sharp=12.0, norm=norm)
        check(c, Run(c)())


def test_rows_outside_the_trees_and_wide_strides():
    c = DiffCase(8, 2, BF16, 32, [(70, 2), (0, 40)], seed=6, q_ld=8 * HD + 24, base_gap=5)
    bits = Run(c)()
    assert (bits[:5] == 0x1234).all()
    check(c, bits)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("seqs", [[(40, 4)], [(40, 1)], [(21, 60)], [(5, 200)]])
def test_what_a_row_does_not_see_does_not_reach_it(seqs, dtype):
    """Infinite and NaN keys and values in the last rows of a sequence: rows in front of them keep their bits."""
    c = DiffCase(8, 4, dtype, 16, seqs, seed=7)
    clean = Run(c)()
    (P, M), inf = seqs[0], 0x7C00 if dtype == F16 else 0x7F80
    n = P + M
    for bad in (inf, inf | 0x8000, inf | 1):
        r = Run(c)
        pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * HD)
        for j in (n - 1, n - 2) if M > 2 else (n - 1,):
            b, t = c.block_list[int(c.trees["table"][0]) + j // c.bt], j % c.bt
            pool[b, :, 0, t * HD + 5] = bad
            v = pool[b, :, 1].reshape(c.Hkv, c.bt // 16, HD, 16)
            v[:, t // 16, 3, t % 16] = bad
        r.pool = dev(pool.reshape(-1))
        bits = r()
        keep = M - (2 if M > 2 else 1)
        assert (bits[:keep] == clean[:keep]).all(), bad
        last = ob.to_f32(bits[M - 1:, :c.H * HD], dtype)
        assert not np.isfinite(last).all()                           # the row itself shows it


def test_an_infinite_value_reaches_the_rows_that_see_it():
    """With finite scores: dim 3 of the pair's output is infinite before the norm, which makes the norm's factor 0."""
    c = DiffCase(4, 2, F16, 16, [(20, 6)], seed=8, norm=False)
    clean = ob.to_f32(Run(c)(), F16)
    r = Run(c)
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * HD)
    j = 23                                                            # the key of the tree's row 3
    b, t = c.block_list[j // 16], j % 16
    pool[b, 0, 1].reshape(1, HD, 16)[0, 3, t] = 0x7C00
    r.pool = dev(pool.reshape(-1))
    got = ob.to_f32(r(), F16)
    col = np.zeros(4 * HD, bool)
    col[[3, 2 * HD + 3]] = True                                      # dim 3 of each query pair's output
    assert (got[:3] == clean[:3]).all() and (got[:, ~col] == clean[:, ~col]).all()
    assert not np.isfinite(got[3:, col]).any()


@pytest.mark.parametrize("seqs,workgroups", [([(40, 1)], None), ([(40, 4)], None), ([(300, 3)], 4096), ([(10, 90)], None), ([(700, 40)], 2048)])
def test_a_key_of_nan_shows_in_every_row_that_sees_it(seqs, workgroups):
    """The first key, alone in its part's first unit for no row: every row and every pair whose map it is in."""
    c = DiffCase(8, 4, BF16, 16, seqs, seed=15)
    r = Run(c, workgroups=workgroups, cut_batch=workgroups is not None)
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * HD)
    pool[c.block_list[int(c.trees["table"][0])], 1, 0, 5] = 0x7FC0     # K of KV head 1, key 0: the second map of the first KV pair
    r.pool = dev(pool.reshape(-1))
    got = ob.to_f32(r()[:, :8 * HD], BF16).reshape(c.n_rows, 4, 2 * HD)
    assert np.isnan(got[:, :2]).all() and np.isfinite(got[:, 2:]).all()


def test_a_second_pass_and_another_stream_give_the_same_bits():
    c = DiffCase(16, 4, BF16, 16, [(900, 1), (300, 1), (77, 1)], seed=9)
    r = Run(c, workgroups=4096)
    first = r()
    r.O.fill_(0x1234)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r.dp.run(r.Q, r.pool, r.O)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert (r.bits() == first).all()


def test_a_captured_pass_follows_the_records_it_reads():
    """Open-ended tiles in a graph: the trees' lengths move on between replays, as esp_chain_advance moves them."""
    lens = [(30, 1), (100, 1), (15, 1)]
    steps = 5
    full = DiffCase(8, 4, F16, 16, [(P + steps, 1) for P, _ in lens], seed=10)
    full.trees["P"] -= steps
    full.seqs = lens
    r = Run(full, open_ended=True)
    g = torch.cuda.CUDAGraph()
    r()
    with torch.cuda.graph(g):
        r.dp.run(r.Q, r.pool, r.O)
    trees = full.trees.copy()
    for s in range(steps):
        full.trees["P"] = trees["P"] + s
        full.seqs = [(int(P), 1) for P in full.trees["P"]]
        r.dp.trees.copy_(device.to_dev(full.trees))
        r.O.fill_(0x1234)
        g.replay()
        torch.cuda.synchronize()
        replayed = r.bits()
        check(full, replayed)
        r.O.fill_(0)
        r.dp.run(r.Q, r.pool, r.O)
        torch.cuda.synchronize()
        assert (r.bits()[:, :8 * HD] == replayed[:, :8 * HD]).all()


def test_the_append_that_the_library_has_serves_it():
    """Rows through esp_attn_prep with a row table, then the attention: as the rows it wrote, read back by esp_kv_gather."""
    from espetero_amd import synth
    device.init(0)
    H, Hkv, n = 8, 4, 24
    pp, a = synth.make_prep("omni", H, Hkv, HD, BF16, n, seed=3, bt=16)
    a["pos"][:, :3] = np.arange(n)[:, None]
    table = np.full((n, 4), -1, np.int32)
    blocks = np.array([2, 0], np.int32)
    table[:, 0], table[:, 1] = blocks[np.arange(n) // 16], np.arange(n) % 16
    pool = torch.zeros(3 * 2 * 16 * Hkv * HD, dtype=torch.int16, device="cuda")
    Q = torch.zeros(n, H * HD, dtype=torch.int16, device="cuda")
    device.attn_prep(pp, *[dev(a[k]) if a[k] is not None else None for k in ("X", "qn_w", "kn_w", "pos", "inv_freq", "rope_sel")], Q, None, None, dev(table),
                     pool, n)
    c = DiffCase(H, Hkv, BF16, 16, [(0, n)], seed=4)
    c.scale = 1.0                                                     # the prep has scaled the queries
    p = c.params()
    K, V = (torch.zeros(n, Hkv * HD, dtype=torch.int16, device="cuda") for _ in range(2))
    device.kv_gather(p, pool, dev(blocks), n, K, V)
    torch.cuda.synchronize()
    u16 = lambda t: t.cpu().numpy().view(np.uint16)  # noqa: E731
    c.Q, c.K, c.V = u16(Q), [u16(K).reshape(n, Hkv, HD)], [u16(V).reshape(n, Hkv, HD)]
    c.pool, c.block_list, c.n_blocks = u16(pool), blocks, 3
    check(c, Run(c)())


def test_a_long_cache_past_32_bit_offsets():
    """A region of 2^31 elements and more in front of the sequence's own blocks: only those are written."""
    device.init(0)
    H, Hkv, bt = 4, 2, 16
    block = 2 * bt * Hkv * HD
    far = (1 << 31) // block + 5
    c = DiffCase(H, Hkv, F16, bt, [(50, 1), (20, 30)], seed=11)
    r = Run(c)
    want = r()
    pool = torch.empty((far + c.n_blocks) * block, dtype=torch.int16, device="cuda")
    pool[far * block:].copy_(r.pool)
    r.dp.blocks += far
    r.pool = pool
    r.O.fill_(0x1234)
    assert (r() == want).all()
    r.dp.blocks -= far
    r.p.kv_base = far * block
    r.O.fill_(0x1234)
    assert (r() == want).all()
    del pool


def test_two_graphs_with_a_workspace_each():
    cases = [DiffCase(8, 2, F16, 16, [(700, 1), (400, 1)], seed=s) for s in (12, 13)]
    runs = [Run(c, workgroups=4096) for c in cases]
    eager = [r() for r in runs]
    graphs = []
    for r in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r.dp.run(r.Q, r.pool, r.O)
        graphs.append(g)
    for _ in range(3):
        for r in runs:
            r.O.fill_(0x1234)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all((r.bits() == e).all() for r, e in zip(runs, eager))


def test_the_workspace_is_checked():
    c = DiffCase(8, 2, F16, 16, [(700, 1)], seed=14)
    r = Run(c, workgroups=4096)
    assert r.parts > 1
    need = abi.attn_lib().esp_attn_diff_workspace_bytes(C.byref(r.p), r.parts)
    r.dp.workspace = torch.empty(need - 1, dtype=torch.uint8, device="cuda")
    with pytest.raises(abi.EspError, match="workspace"):
        r()
