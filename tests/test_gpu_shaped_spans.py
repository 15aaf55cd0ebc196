"""esp_attn_shaped on the device: spans of any numbers, slopes of either sign, windows and rings, at random."""
import random

import numpy as np
import pytest

from shaped_precision import bound
from shaped_utils import ShapedCase
from test_gpu_shaped import MARK, Run
from espetero_amd import abi
from oracle import binding as ob

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16
LEAST, MOST = -2**31, 2**31 - 1


def any_span(rng, P, M, m):
    n = P + M
    near = lambda: rng.choice([rng.randint(0, n), P + m, P + m + 1, P + m - 1, rng.randint(-5, 5), n, n - 1, 16 * rng.randint(0, n // 16)])  # noqa: E731
    far = lambda: rng.choice([LEAST, LEAST + 1, -1, MOST, MOST - 1, n + 1, 10 * n, -10 * n])  # noqa: E731
    return [near() if rng.random() < 0.8 else far() for _ in range(2)]


@pytest.mark.parametrize("seed", range(24))
def test_any_spans(seed):
    rng = random.Random(seed)
    hd = rng.choice([128, 256])
    Hkv = rng.choice([1, 2, 3])
    G = rng.choice([1, 2, 4, 8])
    seqs = [(rng.choice([0, rng.randint(0, 60), rng.randint(0, 500)]), rng.choice([1, rng.randint(1, 8), rng.randint(1, 60)])) for _ in range(rng.randint(1, 3))]
    window = rng.choice([0, 0, rng.randint(1, 300)])
    ring = window > 0 and rng.random() < 0.5
    spans = [[any_span(rng, P, M, m) for m in range(M)] for P, M in seqs]
    if ring:                                                           # keys that lie in front of the ring are nobody's
        spans = [[[max(f, 0), min(e, P + M)] for f, e in s] for s, (P, M) in zip(spans, seqs)]
    c = ShapedCase(Hkv * G, Hkv, hd, rng.choice([F16, BF16]), rng.choice([16, 32]), seqs, window=window, ring=ring, cap=rng.choice([0.0, 0.5, 30.0]),
                   bias=True, spans=spans, sharp=rng.choice([0.3, 1.0, 3.0]), seed=seed)
    c.slopes[:] = np.random.default_rng(seed).choice([0.0, 1.0, -0.02, 1e-3, 30.0, -1e-30], Hkv * G)
    for plan in ({}, dict(workgroups=4096, cut_batch=True), dict(workgroups=1)):
        r = Run(c, **plan)
        bits = r()
        want, tol, which = bound(c, 7)
        got = ob.to_f32(bits[which][:, :c.H * hd], c.dtype).astype(np.float64).reshape(want.shape)
        print(f"  of the bound: {np.max(np.abs(got - want) / np.maximum(tol, 1e-30)):.3f}", flush=True)
        assert np.all(np.abs(got - want) <= tol)
        rest = np.ones(c.n_rows, bool)
        rest[which] = False
        assert (bits[rest] == MARK).all()
