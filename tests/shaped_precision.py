"""Attention with shaped scores: how far an output may be off where a weight enters its product as the sum of two 16-bit numbers."""
import numpy as np

from shaped_utils import HALF
from espetero_amd import abi
from oracle import binding as ob


def bound(c, shift=0, rows=None):
    """(O, how far from it an output may be) in float64, [rows][H][hd].

    Scores and sums are off as in ShapedCase.expected: a weight by 2 e of itself, e = 2^-24 (its products, its operations, its distance to
    the row's reference), sums over n keys by 1.5 n 2^-24. Two numbers of the storage type, each off by half a step u of what
    it stands for, leave u^2 of the weight; in fp16 the second has no step below 2^-24, which leaves 2^-25 of a weight that is 2^shift
    at the row's reference. The reference is no higher than the row's largest score, so that beside the sum of the weights
    taken from that one it is no more than n of those. The output is rounded once."""
    G, hd, u = c.H // c.Hkv, c.hd, HALF[c.dtype]
    step = 2.0 ** (-25 - shift) if c.dtype == abi.ESP_F16 else 0.0
    f = lambda x: ob.to_f32(x, c.dtype).astype(np.float64)  # noqa: E731
    Q = f(c.Q)[:, :c.H * hd].reshape(-1, c.H, hd)
    O, tol, which = [], [], []
    for i, (P, M) in enumerate(c.seqs):
        K, V, base = f(c.K[i]), f(c.V[i]), int(c.trees["base"][i])
        for m in (range(M) if rows is None else [m for m in rows if m < M]):
            lo, end = c.seen(i, m)
            n, ago = end - lo, np.abs(P + m - np.arange(lo, end))
            which.append(base + m)
            for h in range(c.H):
                if n == 0:                                             # a row that sees nothing
                    O.append(np.zeros(hd))
                    tol.append(np.zeros(hd))
                    continue
                k, v, q = K[lo:end, h // G], V[lo:end, h // G], Q[base + m, h]
                x = k @ q * c.scale
                e = (hd + 4) * c.scale * (np.abs(k) @ np.abs(q)).max()
                if c.cap:
                    e += 8 * c.cap if np.abs(x).max() >= 0.69 * c.cap else 16 * np.abs(x).max()
                    x = c.cap * np.tanh(x / c.cap)
                if c.slopes is not None:
                    b = float(c.slopes[h]) * ago
                    x = x - b
                    near = x > x.max() - 100                           # what weighs anything
                    e += 2 * np.abs(b[near]).max() + 6 * np.abs(x[near]).max()
                else:
                    e += 6 * np.abs(x).max()
                w = np.exp(x - x.max())
                l = w.sum()
                o = w @ v / l
                t = (u * u + 2 * e * 2.0 ** -24 + 1.5 * n * 2.0 ** -24) * (w @ np.abs(v)) / l + 2 * step * np.abs(v).sum(0) / l
                O.append(o)
                tol.append(t + u * (np.abs(o) + t) + 2.0 ** -25)
    shape = (len(which), c.H, hd)
    return np.reshape(O, shape), np.reshape(tol, shape), np.array(which)
