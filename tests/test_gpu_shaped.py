"""esp_attn_shaped on the device against the operator in float64."""
import ctypes as C

import numpy as np
import pytest
import torch

from shaped_utils import ShapedCase, documents
from espetero_amd import abi, device, host
from oracle import binding as ob

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16
MARK = 0x1234


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a).view(np.int16 if a.dtype == np.uint16 else a.dtype)).cuda()


class Run:
    def __init__(self, case, rows_per_tile=None, workgroups=None, cut_batch=False, open_ended=False):
        device.init(0)
        self.case, self.p = case, case.params(rows_per_tile)
        self.tiles, self.jobs, self.parts = case.plan(self.p, workgroups, cut_batch)
        tiles = host.open_ended(self.tiles, case.trees) if open_ended else self.tiles
        self.sp = device.ShapedPass(self.p, device.shape_params(case.cap, dev(case.slopes)), case.trees, tiles, self.jobs, self.parts, case.n_rows,
                                    case.block_list, spans=case.spans, pool_blocks=case.n_blocks)
        self.Q, self.pool = dev(case.Q), dev(case.pool)
        self.O = torch.full((case.n_rows, case.q_ld), MARK, dtype=torch.int16, device="cuda")
        print(f"shaped H{case.H}/{case.Hkv} hd{case.hd} bt{case.bt} seqs{case.seqs[:6]} window{case.window} ring{case.ring} cap{case.cap} "
              f"rows{self.p.rows_per_tile} tiles{len(tiles)} parts{self.parts}", flush=True)

    def enqueue(self, stream=None):
        self.sp.run(self.Q, self.pool, self.O, stream=stream)

    def __call__(self):
        self.enqueue()
        torch.cuda.synchronize()
        return self.bits()

    def bits(self):
        return self.O.cpu().numpy().view(np.uint16).copy()


def check(case, bits):
    want, tol = case.expected()
    w = case.H * case.hd
    live = np.isfinite(want[:, 0])
    got = ob.to_f32(bits[:, :w], case.dtype).astype(np.float64)
    worst = np.max(np.abs(got[live] - want[live]) / np.maximum(tol[live], 1e-30))
    print(f"  of the bound: {worst:.3f}", flush=True)
    assert np.all(np.abs(got[live] - want[live]) <= tol[live]), worst
    assert (bits[~live] == MARK).all() and (bits[:, w:] == MARK).all()


SHAPES = [(0.0, False), (20.0, False), (0.0, True), (30.0, True)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cap,bias", SHAPES)
@pytest.mark.parametrize("heads,hd", [((4, 2), 128), ((8, 1), 128), ((32, 1), 128), ((20, 1), 128), ((4, 2), 256), ((16, 1), 256), ((3, 3), 256),
                                      ((40, 1), 128), ((24, 1), 256), ((128, 1), 128)])
def test_single_tokens(heads, hd, cap, bias, dtype):
    c = ShapedCase(*heads, hd, dtype, 16, [(0, 1), (1, 1), (15, 1), (16, 1), (130, 1), (700, 1)], cap=cap, bias=bias, seed=heads[0])
    check(c, Run(c)())
    check(c, Run(c, workgroups=4096)())                              # cut as finely as the planner will


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cap,bias", SHAPES[1:])
@pytest.mark.parametrize("heads,hd,rows", [((4, 4), 128, 5), ((8, 2), 128, 8), ((4, 4), 256, 16), ((8, 2), 256, 4), ((4, 2), 128, 16)])
def test_drafts(heads, hd, rows, cap, bias, dtype):
    c = ShapedCase(*heads, hd, dtype, 64, [(0, rows), (30, rows - 1), (200, rows), (33, 1)], cap=cap, bias=bias, seed=rows)
    check(c, Run(c)())
    check(c, Run(c, workgroups=4096)())
    check(c, Run(c, rows_per_tile=1)())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cap,bias", SHAPES)
@pytest.mark.parametrize("heads,hd,seqs", [((2, 1), 128, [(0, 300)]), ((8, 2), 128, [(50, 133), (0, 17), (7, 64)]), ((4, 4), 128, [(129, 130)]),
                                           ((2, 2), 256, [(0, 129), (31, 127)]), ((8, 1), 256, [(13, 60)]), ((64, 1), 128, [(40, 9), (0, 3)])])
def test_prompts_and_chunks(heads, hd, seqs, cap, bias, dtype):
    c = ShapedCase(*heads, hd, dtype, 16, seqs, cap=cap, bias=bias, seed=3)
    check(c, Run(c)())
    check(c, Run(c, workgroups=2048, cut_batch=True)())


@pytest.mark.parametrize("ring", [False, True])
@pytest.mark.parametrize("window", [1, 16, 100])
@pytest.mark.parametrize("hd,seqs", [(128, [(0, 1), (99, 1), (100, 1), (431, 1)]), (256, [(0, 3), (200, 4)]), (128, [(0, 90), (150, 140)]),
                                     (256, [(170, 100)])])
def test_windows(hd, seqs, window, ring):
    c = ShapedCase(8, 4, hd, F16, 16, seqs, window=window, ring=ring, cap=25.0, bias=True, seed=window)
    check(c, Run(c)())
    check(c, Run(c, workgroups=2048)())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("percent", [0, 50, 100])
def test_documents_and_prefixes(percent, window, hd, dtype):
    seqs = [(0, 330), (77, 150), (200, 3), (90, 1)]
    spans = [documents(0, 330, [0, 1, 64, 200, 201, 329], percent), documents(77, 150, [0, 100], percent), documents(200, 3, [0, 201], percent),
             documents(90, 1, [0, 17], percent)]
    c = ShapedCase(4, 2, hd, dtype, 16, seqs, window=window, spans=spans, cap=30.0, bias=True, seed=percent)
    check(c, Run(c)())
    check(c, Run(c, workgroups=2048, cut_batch=True)())
    check(c, Run(c, rows_per_tile=1)())


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("rows_per_tile", [None, 1, 4])
def test_spans_of_any_numbers_and_rows_that_see_nothing(hd, rows_per_tile):
    big = 2 ** 31 - 1
    some = [(-big - 1, 0), (0, big), (big, 0), (big, big), (5, -7), (50, 55), (70, 20), (0, -big), (54, 1), (3, 100)]
    seqs = [(50, 10), (0, 10), (300, 60)]
    far = [(some[i % 10][0], some[i % 10][1]) if i % 3 else (400, 0) for i in range(60)]
    c = ShapedCase(4, 2, hd, F16, 16, seqs, spans=[some, some, far], cap=0.0, bias=True, seed=5)
    for workgroups in (None, 2048):
        bits = Run(c, rows_per_tile=rows_per_tile, workgroups=workgroups, cut_batch=workgroups is not None)()
        check(c, bits)
        assert (bits[[2, 3]] == 0).all()


def cut(r, each):
    """Run r's pass with every tile in parts of `each` stages of 32 keys, cached ones and the pass's own alike."""
    c, p = r.case, r.p
    tiles, jobs, parts = [], [], 0
    for i, (base, P, table, M) in enumerate(c.trees.tolist()):
        for m in range(0, M, p.rows_per_tile):
            lo = max(0, P + m - c.window + 1) // 16 * 16 if c.window else 0
            hi = P + min(M, m + p.rows_per_tile)
            n = -(-(hi - lo) // (32 * each))
            if n > 1:
                jobs.append((base + m, min(M - m, p.rows_per_tile), parts, n))
            for k in range(n):
                x, y, end = lo + 32 * each * k, lo + 32 * each * (k + 1), k + 1 == n
                last = 1 if end else y - P + 1 if y > P else 0
                tiles.append((i, base + m, min(x, P), P if end else min(y, P), parts + k if n > 1 else -1, last, max(0, x - P), 0))
            parts += n if n > 1 else 0
    tiles, jobs = np.array(tiles, abi.TILE_DT), np.array(jobs, abi.COMBINE_DT) if jobs else np.zeros(0, abi.COMBINE_DT)
    device.validate(p, tiles, c.trees, jobs, parts, c.n_rows, c.block_list, c.n_blocks, shaped=True)
    r.sp.tiles, r.sp.n_tiles, r.sp.jobs, r.sp.n_jobs, r.sp.n_parts = device.to_dev(tiles), len(tiles), device.to_dev(jobs) if len(jobs) else None, len(jobs), parts
    nbytes = abi.attn_lib().esp_attn_shaped_workspace_bytes(C.byref(p), parts)
    r.sp.workspace = torch.full((max(nbytes, 16),), 0xff, dtype=torch.uint8, device="cuda")    # NaN: nothing is merged that was not written
    return r


@pytest.mark.parametrize("hd,heads", [(128, (8, 2)), (256, (4, 2)), (128, (7, 1))])
@pytest.mark.parametrize("window,ring", [(0, False), (60, False), (60, True)])
@pytest.mark.parametrize("each", [1, 2, 5])
def test_any_parts(each, window, ring, hd, heads):
    """Parts that some rows, or all, see nothing of among them: spans leave them other keys."""
    seqs = [(100, 70), (0, 90), (31, 20), (16, 40)] if not ring else [(100, 20), (0, 24), (31, 20)]
    spans = [documents(P, M, [0, 40, 64, 80], 50) if i % 2 == 0 else [(3, P + M)] * M for i, (P, M) in enumerate(seqs)]
    for sp in (None, spans):
        c = ShapedCase(*heads, hd, BF16, 16, seqs, window=window, ring=ring, spans=sp, cap=20.0, bias=True, seed=19)
        check(c, cut(Run(c), each)())


def test_sharp_softmax_and_large_caps():
    for cap in (0.0, 1.0, 200.0):
        c = ShapedCase(8, 2, 128, F16, 16, [(500, 1), (90, 3), (60, 70)], seed=5, sharp=12.0, cap=cap)
        check(c, Run(c)())


@pytest.mark.parametrize("cap", [2.0 ** 120, 1e30, 1e12, 1e8, 1e5, 1000.0, 0.1, 1e-4, 1e-12])
def test_caps_far_from_the_scale(cap):
    """Of a cap far above the scores nothing is left but the scores, of one far below their signs."""
    for hd, seqs in ((128, [(300, 1), (40, 3)]), (256, [(90, 60), (0, 33)]), (128, [(50, 150)])):
        c = ShapedCase(8, 2, hd, F16, 16, seqs, seed=18, cap=cap, bias=hd == 256)
        check(c, Run(c)())


def test_rows_outside_the_trees_and_wide_strides():
    for hd in (128, 256):
        c = ShapedCase(8, 2, hd, BF16, 32, [(70, 2), (0, 40)], seed=6, q_ld=8 * hd + 24, base_gap=5, cap=10.0)
        check(c, Run(c)())


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("seqs", [[(40, 4)], [(40, 1)], [(21, 60)], [(5, 200)]])
def test_what_a_row_does_not_see_does_not_reach_it(seqs, dtype, hd, cap):
    """Infinite and NaN keys and values in the last rows of a sequence: rows in front of them keep their bits."""
    c = ShapedCase(8, 4, hd, dtype, 16, seqs, seed=7, cap=cap)
    clean = Run(c)()
    (P, M), inf = seqs[0], 0x7C00 if dtype == F16 else 0x7F80
    n = P + M
    for bad in (inf, inf | 0x8000, inf | 1):
        r = Run(c)
        pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * hd)
        for j in (n - 1, n - 2) if M > 2 else (n - 1,):
            b, t = c.block_list[int(c.trees["table"][0]) + j // c.bt], j % c.bt
            pool[b, :, 0, t * hd + 5] = bad
            v = pool[b, :, 1].reshape(c.Hkv, c.bt // 16, hd, 16)
            v[:, t // 16, 3, t % 16] = bad
        r.pool = dev(pool.reshape(-1))
        bits = r()
        keep = M - (2 if M > 2 else 1)
        assert (bits[:keep] == clean[:keep]).all(), bad
        assert not np.isfinite(ob.to_f32(bits[M - 1:], dtype)).all()  # the row itself shows it


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("what", ["K", "V"])
@pytest.mark.parametrize("rows", [6, 150])
def test_another_document_does_not_reach_a_row(rows, what, hd):
    """NaN in the whole of the first document: the rows of the second keep their bits, and keys behind the last are never read as numbers."""
    P = 45
    spans = [documents(P, rows, [0, P + 3])]
    c = ShapedCase(4, 2, hd, BF16, 16, [(P, rows)], spans=spans, seed=8, cap=20.0, bias=True)
    clean = Run(c)()
    check(c, clean)
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * hd)
    for j in range(P + 3):
        b, t = c.block_list[j // 16], j % 16
        if what == "K":
            pool[b, :, 0, t * hd:(t + 1) * hd] = 0x7FC0
        else:
            pool[b, :, 1].reshape(c.Hkv, 1, hd, 16)[:, 0, :, t] = 0x7FC0
    r = Run(c)
    r.pool = dev(pool.reshape(-1))
    bits = r()
    assert (bits[3:] == clean[3:]).all()
    assert np.isnan(ob.to_f32(bits[:3], BF16)).all()


def test_an_infinite_value_reaches_the_rows_that_see_it():
    c = ShapedCase(4, 2, 128, F16, 16, [(20, 6)], seed=8, bias=True)
    clean = ob.to_f32(Run(c)(), F16)
    r = Run(c)
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * 128)
    j = 23                                                            # the key of the tree's row 3
    b, t = c.block_list[j // 16], j % 16
    pool[b, 0, 1].reshape(1, 128, 16)[0, 3, t] = 0x7C00
    r.pool = dev(pool.reshape(-1))
    got = ob.to_f32(r(), F16)
    col = np.zeros(4 * 128, bool)
    col[[3, 128 + 3]] = True                                          # dim 3 of the KV head's two query heads
    assert (got[:3] == clean[:3]).all() and (got[:, ~col] == clean[:, ~col]).all()
    assert (got[3:, col] == np.inf).all()


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("seqs,workgroups", [([(40, 1)], None), ([(40, 4)], None), ([(300, 3)], 4096), ([(10, 90)], None), ([(700, 40)], 2048)])
def test_a_key_of_nan_shows_in_every_row_that_sees_it(seqs, workgroups, cap):
    c = ShapedCase(8, 4, 128, BF16, 16, seqs, seed=15, cap=cap)
    r = Run(c, workgroups=workgroups, cut_batch=workgroups is not None)
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * 128)
    pool[c.block_list[int(c.trees["table"][0])], 1, 0, 5] = 0x7FC0     # K of KV head 1, key 0
    r.pool = dev(pool.reshape(-1))
    got = ob.to_f32(r(), BF16).reshape(c.n_rows, 8, 128)
    assert np.isnan(got[:, 2:4]).all() and np.isfinite(np.delete(got, [2, 3], 1)).all()


def test_a_cap_holds_infinite_scores():
    """A key whose products are beyond fp32: the cap of its score, not NaN."""
    c = ShapedCase(2, 1, 128, BF16, 16, [(20, 1), (20, 60)], seed=16, cap=5.0)
    for i in range(2):
        c.K[i][7] = 0x7F00                                             # 2^127 in every dim
    pool = c.pool.reshape(c.n_blocks, c.Hkv, 2, c.bt * 128)
    for t in c.trees["table"]:
        pool[c.block_list[int(t)], :, 0, 7 * 128:8 * 128] = 0x7F00
    c.Q[:] = np.abs(c.Q.view(np.int16)).view(np.uint16) & 0x7FFF       # one sign: the sum is infinite, not inf - inf
    got = ob.to_f32(Run(c)(), BF16).astype(np.float64)
    for i, (P, M) in enumerate(c.seqs):
        for m in range(M):
            lo, end = c.seen(i, m)
            K, V = (ob.to_f32(x[i], BF16).astype(np.float64)[lo:end, 0] for x in (c.K, c.V))
            for h in range(2):
                r = int(c.trees["base"][i]) + m
                x = 5 * np.tanh(K @ ob.to_f32(c.Q, BF16).astype(np.float64)[r, h * 128:(h + 1) * 128] * c.scale / 5)
                w = np.exp(x - x.max())
                o = w @ V / w.sum()
                assert np.abs(got[r, h * 128:(h + 1) * 128] - o).max() <= 2.0 ** -6.5 * np.abs(V).max()


def test_a_second_pass_and_another_stream_give_the_same_bits():
    c = ShapedCase(16, 4, 128, BF16, 16, [(900, 1), (300, 1), (77, 1)], seed=9, cap=50.0, bias=True)
    r = Run(c, workgroups=4096)
    first = r()
    r.O.fill_(MARK)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    r.enqueue(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert (r.bits() == first).all()


def test_a_captured_pass_follows_the_records_it_reads():
    """Open-ended tiles in a graph: the trees' lengths move on between replays, as esp_chain_advance moves them; spans stay."""
    steps = 5
    lens = [(30, 1), (100, 1), (15, 1)]
    full = ShapedCase(8, 4, 128, F16, 16, [(P + steps, 1) for P, _ in lens], seed=10, cap=20.0, bias=True, spans=[[(4, 20)], [(0, 0)], [(15, 0)]])
    full.trees["P"] -= steps
    full.seqs = lens
    r = Run(full, open_ended=True)
    g = torch.cuda.CUDAGraph()
    r()
    with torch.cuda.graph(g):
        r.enqueue()
    trees = full.trees.copy()
    for s in range(steps):
        full.trees["P"] = trees["P"] + s
        full.seqs = [(int(P), 1) for P in full.trees["P"]]
        r.sp.trees.copy_(device.to_dev(full.trees))
        r.O.fill_(MARK)
        g.replay()
        torch.cuda.synchronize()
        replayed = r.bits()
        check(full, replayed)
        r.O.fill_(0)
        r.enqueue()
        torch.cuda.synchronize()
        assert (r.bits() == replayed).all()


def test_without_shapes_it_is_the_plain_attention():
    """The operator of esp_attn_forward's: within both kernels' roundings of each other, tiled and streaming."""
    for seqs in ([(500, 1), (60, 1)], [(130, 200)]):
        c = ShapedCase(8, 2, 128, F16, 16, seqs, seed=17)
        got = ob.to_f32(Run(c)(), F16)
        p = c.params()
        p.rows_per_tile = 128 if seqs[0][1] > 1 else 1
        resident, groups = device.plan_hint(p)
        tiles, jobs, parts = host.plan_tiles(c.trees, groups, 0, None, host.options_mi355x(p.rows_per_tile, resident))
        K, V = (np.concatenate([x[i][P:].reshape(M, -1) for i, (P, M) in enumerate(seqs)]) for x in (c.K, c.V))
        dp = device.DevicePass(p, c.trees, tiles, jobs, parts, c.n_rows, c.block_list, pool_blocks=c.n_blocks)
        O = torch.zeros(c.n_rows, 8 * 128, dtype=torch.int16, device="cuda")
        dp.run(dev(c.Q), dev(K), dev(V), dev(c.pool), O)
        torch.cuda.synchronize()
        want = ob.to_f32(O.cpu().numpy().view(np.uint16), F16)
        _, tol = c.expected()
        assert (np.abs(got - want) <= 2 * tol).all()


def test_a_long_cache_past_32_bit_offsets():
    """A region of 2^31 elements and more in front of the sequence's own blocks: only those are written."""
    device.init(0)
    H, Hkv, bt, hd = 4, 2, 16, 128
    block = 2 * bt * Hkv * hd
    far = (1 << 31) // block + 5
    c = ShapedCase(H, Hkv, hd, F16, bt, [(50, 1), (20, 30)], seed=11, cap=20.0)
    for rows in (None, 1):
        r = Run(c, rows_per_tile=rows)
        want = r()
        pool = torch.empty((far + c.n_blocks) * block, dtype=torch.int16, device="cuda")
        pool[far * block:].copy_(r.pool)
        r.sp.blocks += far
        r.pool = pool
        r.O.fill_(MARK)
        assert (r() == want).all()
        r.sp.blocks -= far
        r.sp.params.kv_base = far * block
        r.O.fill_(MARK)
        assert (r() == want).all()
        del pool


def test_two_graphs_with_a_workspace_each():
    cases = [ShapedCase(8, 2, 128, F16, 16, [(700, 1), (400, 1)], seed=s, cap=30.0) for s in (12, 13)]
    runs = [Run(c, workgroups=4096) for c in cases]
    eager = [r() for r in runs]
    graphs = []
    for r in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r.enqueue()
        graphs.append(g)
    for _ in range(3):
        for r in runs:
            r.O.fill_(MARK)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all((r.bits() == e).all() for r, e in zip(runs, eager))


def test_the_workspace_is_checked():
    c = ShapedCase(8, 2, 128, F16, 16, [(700, 1)], seed=14)
    r = Run(c, workgroups=4096)
    assert r.parts > 1
    need = abi.attn_lib().esp_attn_shaped_workspace_bytes(C.byref(r.p), r.parts)
    r.sp.workspace = torch.empty(need - 1, dtype=torch.uint8, device="cuda")
    with pytest.raises(abi.EspError, match="workspace"):
        r()
