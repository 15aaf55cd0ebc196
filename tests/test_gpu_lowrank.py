"""esp_lowrank_add on the device against the operator in float64."""
import numpy as np
import pytest
import torch

from espetero_amd import abi, device, synth
from oracle import binding as ob

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16


class Case:
    def __init__(self, adapter, D, rank, slices, dtype, n_adapters, seed=0, x_ld=None, y_ld=None, x_scale=1.0):
        rng = np.random.default_rng(seed)
        self.adapter = np.asarray(adapter, np.int32)
        self.D, self.rank, self.slices, self.dtype, self.na = D, rank, slices, dtype, n_adapters
        n, S, W = len(self.adapter), len(slices), sum(w for _, w in slices)
        self.x_ld = x_ld or D
        self.y_ld = y_ld or max(o + w for o, w in slices)
        bits = lambda x: synth._bits(x, dtype)  # noqa: E731
        self.X = bits(rng.standard_normal((n, self.x_ld), dtype=np.float32) * x_scale)
        self.A = bits(rng.standard_normal((n_adapters, S * rank, D), dtype=np.float32) * D ** -0.5)
        self.B = bits(rng.standard_normal((n_adapters, W, rank), dtype=np.float32) * 0.5)
        self.scale = rng.uniform(0.5, 2.0, n_adapters).astype(np.float32)
        self.Y = rng.standard_normal((n, self.y_ld), dtype=np.float32)

    def expected(self):
        """(Y, how far off a kernel may be). An intermediate is off by (D + 16) 2^-24 of its products' sum (fp32, D products, up to 16
        splits) and by 2^-23 of the row's largest where it becomes 16-bit terms; the second sum by (4 rank) 2^-24 of its own; the
        factor, the addition and the store by 2^-22 of the result's parts."""
        f = lambda x: ob.to_f32(x, self.dtype).astype(np.float64)  # noqa: E731
        X, A, B = f(self.X)[:, :self.D], f(self.A), f(self.B)
        Y, tol = self.Y.astype(np.float64), np.zeros(self.Y.shape)
        for r, a in enumerate(self.adapter):
            if a < 0:
                continue
            at = 0
            for s, (off, w) in enumerate(self.slices):
                As = A[a, s * self.rank:(s + 1) * self.rank]
                Bs = B[a, at:at + w]
                low, mag = As @ X[r], np.abs(As) @ np.abs(X[r])
                e = (self.D + 16) * 2.0 ** -24 * mag + 2.0 ** -23 * np.abs(low).max()
                add, size = Bs @ low, np.abs(Bs) @ np.abs(low)
                c = float(self.scale[a])
                tol[r, off:off + w] = c * (np.abs(Bs) @ e + 4 * self.rank * 2.0 ** -24 * size) + 2.0 ** -22 * (np.abs(Y[r, off:off + w]) + c * size)
                Y[r, off:off + w] += c * add
                at += w
        return Y, tol

    def prepare(self):
        device.init(0)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int16 if a.dtype == np.uint16 else a.dtype).copy()).cuda()  # noqa: E731
        self.p = device.lowrank_params(self.D, self.rank, self.slices, self.dtype, self.x_ld, self.y_ld, self.na)
        self.lp = device.LowRankPass(self.p, self.adapter)
        self.dX, self.dA, self.dB, self.ds, self.dY = (dev(a) for a in (self.X, self.A, self.B, self.scale, self.Y))
        print(f"lowrank rows{len(self.adapter)} D{self.D} rank{self.rank} slices{self.slices} tiles{self.lp.n_tiles} of {self.p.rows_per_tile}", flush=True)
        return self

    def run(self):
        self.lp.run(self.dX, self.dA, self.dB, self.ds, self.dY)

    def check(self):
        self.prepare().run()
        torch.cuda.synchronize()
        got = self.dY.cpu().numpy()
        want, tol = self.expected()
        err = np.abs(got - want)
        print(f"  of the bound: {np.max(err[tol > 0] / tol[tol > 0], initial=0):.3f}", flush=True)
        assert np.all(err <= tol)                                     # 0 where no adapter reaches: the bits stay
        return got


QKV = [(0, 256), (256, 64), (320, 64)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 128])
@pytest.mark.parametrize("adapter", [[0], [1, 0, -1, 2, 1, 1], [2] * 17 + [-1] + [0] * 5])
def test_ranks(adapter, rank, dtype):
    Case(adapter, 256, rank, QKV, dtype, 3, seed=rank).check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [8, 40, 264, 1000, 5120])
def test_widths(D, dtype):
    Case([0, 1, 0], D, 16, QKV, dtype, 2, seed=D).check()


@pytest.mark.parametrize("slices", [[(0, 1)], [(3, 17)], [(7, 300), (320, 5)], [(600, 33), (0, 513)], [(0, 128), (200, 16), (216, 40), (500, 257)]])
def test_slices_of_any_width_and_place(slices):
    for dtype in (F16, BF16):
        Case([1, -1, 0, 0, 1], 128, 16, slices, dtype, 2, seed=1, y_ld=903).check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts", [[1, 0, 15], [16, 17, 1], [31, 64, 65], [130, 3, 257], [700, 1, 40]])
def test_prompts(counts, dtype):
    rng = np.random.default_rng(sum(counts))
    adapter = np.concatenate([np.full(n, a) for a, n in enumerate(counts)] + [np.full(7, -1)])
    Case(adapter, 320, 32, QKV, dtype, 3, seed=2).check()
    Case(rng.permutation(adapter), 320, 8, QKV, dtype, 3, seed=3).check()   # rows of one adapter anywhere in the batch


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,rank,slices,counts,y_ld", [
    (1000, 128, [(7, 300), (320, 5)], [150, 3], 331), (264, 24, [(0, 1)], [130], 1), (40, 64, [(1, 2), (3, 1), (10, 129)], [129, 64, 65], 139),
    (8, 8, [(0, 127), (130, 129)], [200, 1], 261), (512, 16, [(0, 2048), (2048, 513)], [1500, 1400], 2561), (2560, 16, [(5, 260)], [63, 129, 128], 400)])
def test_tiles_of_64_rows(D, rank, slices, counts, y_ld, dtype):
    adapter = np.random.default_rng(D).permutation(np.concatenate([np.full(n, a) for a, n in enumerate(counts)] + [[-1]]))
    Case(adapter, D, rank, slices, dtype, len(counts), seed=D, y_ld=y_ld).check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,rank", [(8, 8), (24, 16), (32, 24), (56, 8), (520, 32), (2048, 16), (4096, 8)])
def test_one_launch_for_little_of_a(D, rank, dtype):
    for adapter in ([0], [1] * 16 + [0] * 3):
        Case(adapter, D, rank, [(3, 1030), (1040, 1), (1050, 17)], dtype, 2, seed=D, y_ld=1067).check()


def test_many_adapters_and_strides():
    rng = np.random.default_rng(0)
    Case(rng.integers(-1, 40, 100), 512, 16, QKV, BF16, 40, seed=4, x_ld=520, y_ld=391).check()


def test_intermediates_outside_the_range_of_fp16():
    for x in (3000.0, 1e-6):
        Case([0, 1, 0, -1], 512, 16, QKV, F16, 2, seed=5, x_scale=x).check()
    for x in (1e20, 1e-20):
        Case([0, 1, 0, -1], 512, 16, QKV, BF16, 2, seed=6, x_scale=x).check()
    for dtype, x in ((F16, 3000.0), (F16, 1e-6), (BF16, 1e20), (BF16, 1e-20)):
        Case([0] * 5, 4096, 16, QKV, dtype, 1, seed=5, x_scale=x).check()
        Case([0, 1] * 70, 512, 16, QKV, dtype, 2, seed=5, x_scale=x).check()


@pytest.mark.parametrize("n,D,rank", [(20, 256, 16), (20, 2048, 40), (150, 256, 16)])
def test_a_row_of_infinities_stays_in_its_row(n, D, rank):
    c = Case([0] * n, D, rank, QKV, BF16, 1, seed=7)
    clean = c.check()
    c.X[3, 7], c.X[11, 9] = 0x7F80, 0x7FC0
    c.prepare().run()
    torch.cuda.synchronize()
    got = c.dY.cpu().numpy()
    keep = [r for r in range(n) if r not in (3, 11)]
    assert (got[keep] == clean[keep]).all()
    assert not np.isfinite(got[3]).any() and np.isnan(got[11]).all()


def test_no_rows_and_no_adapters():
    c = Case([-1, -1], 64, 8, QKV, F16, 1).prepare()
    c.run()
    torch.cuda.synchronize()
    assert (c.dY.cpu().numpy() == c.Y).all()


def test_replays_and_streams_give_the_same_bits():
    c = Case(np.random.default_rng(1).integers(-1, 4, 50), 1024, 16, QKV, BF16, 4, seed=8)
    first = c.check()
    start = torch.from_numpy(c.Y).cuda()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    for _ in range(3):
        c.dY.copy_(start)
        g.replay()
        torch.cuda.synchronize()
        assert (c.dY.cpu().numpy() == first).all()
        c.dY.copy_(start)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c.run()
        side.synchronize()
        assert (c.dY.cpu().numpy() == first).all()
