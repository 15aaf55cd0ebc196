"""How far an output of differential attention may be from the operator in float64 when the weights enter their product with V as two
numbers of the storage type, and the operator with weights of any number of them."""
import numpy as np

from diff_utils import HALF, HD
from espetero_amd import abi, synth
from oracle import binding as ob


def case_rows(c):
    """(output row, pair, [(factor of the map, scores, |K| |q|) of both], V) of every row and pair, in float64."""
    f = lambda x: ob.to_f32(x, c.dtype).astype(np.float64)  # noqa: E731
    Q, G = f(c.Q), c.H // c.Hkv
    for i, (P, M) in enumerate(c.seqs):
        K, V, base = f(c.K[i]), f(c.V[i]), int(c.trees["base"][i])
        for m in range(M):
            n = P + m + 1
            for pair in range(c.H // 2):
                kv, maps = 2 * (pair // G), []
                for e in (0, 1):
                    q = Q[base + m, (2 * pair + e) * HD:(2 * pair + e + 1) * HD]
                    maps.append((1.0 if e == 0 else -float(c.weight[pair]), K[:n, kv + e] @ q * c.scale, np.abs(K[:n, kv + e]) @ np.abs(q) * c.scale))
                yield base + m, pair, maps, np.concatenate([V[:n, kv], V[:n, kv + 1]], -1)


def bound(c, numbers):
    """(O, how far off) without norm and window. numbers: how many 16-bit numbers hold the weights of the first and the second map.

    A weight p of the product is off by u p where one number holds it and by u^2 p where two do, u half a step of the storage type, and by
    no less than half a step of fp16's smallest numbers, 2^-25, in units in which the largest weight is 1 or more. The other terms are
    those of DiffCase.expected, with 3 n 2^-24 for the sums, since two products add up, and 2^-20 for what follows them."""
    assert c.norm_w is None and not c.window
    u = HALF[c.dtype]
    O, tol = np.zeros((c.n_rows, c.H * HD)), np.zeros((c.n_rows, c.H * HD))
    for row, pair, maps, v in case_rows(c):
        n, o, d = len(v), np.zeros(2 * HD), np.zeros(2 * HD)
        for (factor, s, size), k in zip(maps, numbers):
            w = np.exp(s - s.max())
            L = w.sum()
            es = 2.0 ** -24 * (132 * size.max() + 4 * np.abs(s).max() + 8)
            o += factor * (w @ v) / L
            d += abs(factor) * ((u ** k + 2 * es + 3 * n * 2.0 ** -24 + 2.0 ** -20) * (w @ np.abs(v)) + (2.0 ** -25 if c.dtype == abi.ESP_F16 else 0) * np.abs(v).sum(0)) / L
        at = slice(2 * pair * HD, 2 * (pair + 1) * HD)
        O[row, at], d = o * c.factor, d * c.factor
        tol[row, at] = d + u * (np.abs(O[row, at]) + d) + 2.0 ** -25
    return O, tol


def with_weights_of(c, numbers):
    """The operator in float64 but for the weights, relative to the largest, as sums of so many numbers of the storage type, and the output
    in it."""
    to = lambda x: ob.to_f32(synth._bits(x.astype(np.float32), c.dtype), c.dtype).astype(np.float64)  # noqa: E731
    O = np.zeros((c.n_rows, c.H * HD))
    for row, pair, maps, v in case_rows(c):
        o = np.zeros(2 * HD)
        for (factor, s, _), k in zip(maps, numbers):
            w = np.exp(s - s.max())
            held = np.zeros_like(w)
            for _ in range(k):
                held += to(w - held)
            o += factor * (held @ v) / w.sum()
        O[row, 2 * pair * HD:2 * (pair + 1) * HD] = o * c.factor
    return to(O)
