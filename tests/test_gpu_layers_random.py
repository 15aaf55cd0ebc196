"""Linear attention and attention with shaped scores at random shapes, from fixed seeds: every choice that the other tests make one at a time."""
import numpy as np
import pytest

import test_gpu_linear as linear
import test_gpu_linear_segments as segments
import test_gpu_shaped as shaped
from espetero_amd import abi
from linear_utils import LinearCase
from shaped_utils import ShapedCase, documents

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(60))
def test_shaped(seed):
    rng = np.random.default_rng(seed)
    pick = lambda *x: x[rng.integers(len(x))]  # noqa: E731
    hd, dtype, bt = pick(128, 256), pick(abi.ESP_F16, abi.ESP_BF16), pick(16, 32, 64)
    Hkv, G = pick(1, 2, 3), pick(1, 2, 3, 4, 7, 8, 16, 32)
    H = Hkv * G
    few = rng.random() < 0.35
    seqs = []
    for _ in range(rng.integers(1, 5)):
        P = int(pick(0, 1, rng.integers(0, 40), rng.integers(0, 400)))
        seqs.append((P, int(pick(1, rng.integers(1, 5))) if few else int(pick(1, rng.integers(1, 60), rng.integers(1, 200)))))
    window = int(pick(0, 0, rng.integers(1, 300)))
    ring = window > 0 and rng.random() < 0.5
    kind = pick("none", "documents", "any")
    spans = None
    if kind == "documents":
        spans = [documents(P, M, np.unique(np.concatenate([[0], rng.integers(0, P + M, rng.integers(0, 5))])), int(rng.integers(0, 101))) for P, M in seqs]
    elif kind == "any":
        spans = [np.stack([rng.integers(-5, P + M + 5, M), rng.integers(-5, P + M + 5, M)], -1) * rng.integers(0, 2, (M, 1)) for P, M in seqs]
    c = ShapedCase(H, Hkv, hd, dtype, bt, seqs, window=window, ring=ring, cap=float(pick(0.0, 0.0, 2.0, 15.0, 50.0, 1e4)), bias=rng.random() < 0.5, spans=spans,
                   seed=seed, q_ld=H * hd + 8 * int(rng.integers(0, 4)), sharp=float(pick(0.5, 1.0, 5.0)), base_gap=int(rng.integers(0, 3)))
    most = max(M for _, M in seqs)
    rows_per_tile = None if rng.random() < 0.6 else int(rng.integers(1, min(most, 128 // G) + 1))
    r = shaped.Run(c, rows_per_tile=rows_per_tile, workgroups=pick(None, None, 7, 300, 5000))
    if rng.random() < 0.4:
        shaped.cut(r, int(rng.integers(1, 6)))
    shaped.check(c, r())


@pytest.mark.parametrize("seed", range(60))
def test_linear(seed):
    rng = np.random.default_rng(1000 + seed)
    pick = lambda *x: x[rng.integers(len(x))]  # noqa: E731
    dk, dv, dtype = pick(64, 128), pick(64, 128, 192, 256), pick(abi.ESP_F16, abi.ESP_BF16)
    Hk, group = int(pick(1, 2, 3)), int(pick(1, 2, 5))
    n = int(rng.integers(1, 7))
    seqs, slot = [], n
    for i in range(n):
        rows = int(pick(0, 1, rng.integers(1, 9), rng.integers(9, 80), rng.integers(60, 400)))
        to = pick("same", "fork", "fresh", "drop")
        seqs.append((rows, -1 if to == "fresh" else i, i if to == "same" else -1 if to == "drop" else slot + i))
    c = LinearCase(Hk * group, Hk, dk, dv, dtype, seqs, n_states=2 * n, row_decay=rng.random() < 0.5, seed=seed, gap=int(rng.integers(0, 4)),
                   wide=8 * int(rng.integers(0, 4)), decay=pick(None, None, 0.0, -0.5, -20.0), size=float(pick(0.1, 1.0, 8.0)))
    r = linear.Run(c, workgroups=pick(None, 1, 64, 5000))
    if rng.random() < 0.4 and c.n_rows:
        segments.cut(r, int(rng.integers(1, 4)))
    linear.check(c, r())
