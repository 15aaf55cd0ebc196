"""Attention with shaped scores for the tests: small paged cases in the library's pool layout, the operator in float64, and how far a
kernel that rounds as the library says may be from it."""
import numpy as np

from espetero_amd import abi, device, host, synth
from oracle import binding as ob

HALF = {abi.ESP_F16: 2.0 ** -11, abi.ESP_BF16: 2.0 ** -8}     # half a step of the storage type, relative


class ShapedCase:
    """seqs: (cached keys, rows). Rows and cached keys lie in the pool; memory that holds no key is filled with NaN."""

    def __init__(self, H, Hkv, hd, dtype, bt, seqs, window=0, ring=False, cap=0.0, bias=False, spans=None, seed=0, q_ld=None, sharp=1.0, base_gap=0):
        rng = np.random.default_rng(seed)
        self.H, self.Hkv, self.hd, self.dtype, self.bt, self.seqs, self.window = H, Hkv, hd, dtype, bt, list(seqs), window
        bits = lambda x: synth._bits(x, dtype)  # noqa: E731
        nan = np.uint16(0x7E00 if dtype == abi.ESP_F16 else 0x7FC0)
        most = max(M for _, M in seqs)
        self.ring = -(-(window + most) // bt) if ring else 0
        per = [self.ring or -(-(P + M) // bt) for P, M in seqs]
        self.n_blocks = sum(per) + 2
        order = rng.permutation(self.n_blocks).astype(np.int32)
        self.n_rows = base_gap + sum(M for _, M in seqs)
        self.q_ld = q_ld or H * hd
        self.Q = np.full((self.n_rows, self.q_ld), nan, np.uint16)
        self.Q[:, :H * hd] = bits(rng.standard_normal((self.n_rows, H * hd), dtype=np.float32) * np.float32(sharp))
        self.trees = np.zeros(len(seqs), abi.TREE_DT)
        self.pos = np.zeros((self.n_rows, 4), np.int32)
        k_plane = np.full((self.n_blocks, Hkv, bt, hd), nan, np.uint16)
        v_plane = np.full((self.n_blocks, Hkv, bt, hd), nan, np.uint16)
        self.K, self.V, self.block_list = [], [], order
        base, used = base_gap, 0
        for i, ((P, M), nb) in enumerate(zip(seqs, per)):
            n = P + M
            K, V = (bits(rng.standard_normal((n, Hkv, hd), dtype=np.float32)) for _ in range(2))
            self.K.append(K)
            self.V.append(V)
            self.trees[i] = (base, P, used, M)
            self.pos[base:base + M, :3] = (P + np.arange(M))[:, None]
            for j in range(max(0, n - self.ring * bt) if ring else 0, n):
                b = used + (j // bt) % self.ring if ring else order[used + j // bt]
                k_plane[b, :, j % bt], v_plane[b, :, j % bt] = K[j], V[j]
            base += M
            used += nb
        vt = v_plane.reshape(self.n_blocks, Hkv, bt // 16, 16, hd).transpose(0, 1, 2, 4, 3).reshape(self.n_blocks, Hkv, bt * hd)
        self.pool = np.concatenate([k_plane.reshape(self.n_blocks, Hkv, bt * hd), vt], -1).reshape(-1)
        self.cap, self.scale = cap, hd ** -0.5
        self.slopes = np.exp2(-8.0 * (1 + np.arange(H)) / H).astype(np.float32) if bias else None
        self.spans = None
        if spans is not None:                                          # of every sequence: (first, prefix) per row
            self.spans = np.zeros((self.n_rows, 2), np.int32)
            self.spans[base_gap:] = np.concatenate([np.asarray(s, np.int64).reshape(-1, 2) for s in spans])

    def params(self, rows_per_tile=None):
        p = synth.make_params(self.H, self.Hkv, self.hd, self.dtype, self.bt, window=self.window, ring=self.ring, scale=self.scale, rows_per_tile=1)
        p.q_ld = self.q_ld
        p.rows_per_tile = rows_per_tile or device.attn_shaped_rows(p, max(M for _, M in self.seqs))
        return p

    def plan(self, p, workgroups=None, cut_batch=False):
        resident, groups = device.attn_shaped_hint(p) if workgroups is None else (workgroups, p.Hkv)
        o = host.options_mi355x(p.rows_per_tile, resident)
        if cut_batch:
            o.cut_batch, o.min_chunk, o.min_span, o.item_steps, o.part_steps = 1, 32, 32, 1, 0
        return host.plan_tiles(self.trees, groups, self.window, self.pos if self.window else None, o)

    def seen(self, i, m):
        """[first, end) of the keys that row m of sequence i sees."""
        P, M = self.seqs[i]
        q = P + m
        first, end = 0, q + 1
        if self.spans is not None:
            first, prefix = (int(x) for x in self.spans[int(self.trees["base"][i]) + m])
            first, end = max(first, 0), min(max(q + 1, prefix), P + M)
        if self.window:
            first = max(first, q - self.window + 1)
        return first, max(first, end)

    def expected(self):
        """(O, how far from it an output may be) in float64, [n_rows][H * hd] with NaN in rows of no sequence.

        A score is off by e = 2^-24 ((hd + 4) scale max sum |q| |k|, the products' sum and its factor; 6 |x|, the operations on it and its
        distance to the row's reference in log2 units; 16 max |x| for a polynomial within 6 steps and its operations, or where scores of the case come
        to 0.69 caps 8 cap, the cap's exponential, sum, reciprocal and product; 2 |bias|), the weight by a
        factor of 1 + d, |d| <= u + 2 e with u half a step of the storage type for its own rounding; sums over n keys in fp32 add n 2^-24
        (weights half of that again). With A = sum p |v| the output is off by (u + 2 e + 1.5 n 2^-24) A and its rounding u |O|. A row that
        sees nothing gets zeros."""
        G, hd, u = self.H // self.Hkv, self.hd, HALF[self.dtype]
        f = lambda x: ob.to_f32(x, self.dtype).astype(np.float64)  # noqa: E731
        Q = f(self.Q)[:, :self.H * hd].reshape(-1, self.H, hd)
        live = np.isfinite(Q[:, 0, 0])
        largest = max(np.abs(np.einsum("khd,rhd->rkh", np.repeat(f(K), G, 1), np.nan_to_num(Q[live]))).max() for K in self.K) * self.scale if self.cap else 0
        O = np.full((self.n_rows, self.H, hd), np.nan)
        tol = np.full_like(O, np.nan)
        for i, (P, M) in enumerate(self.seqs):
            K, V = f(self.K[i]), f(self.V[i])
            base = int(self.trees["base"][i])
            for m in range(M):
                lo, end = self.seen(i, m)
                r, n = base + m, end - lo
                if n == 0:
                    O[r], tol[r] = 0.0, 0.0
                    continue
                ago = np.abs(P + m - np.arange(lo, end))
                for h in range(self.H):
                    k, v, q = K[lo:end, h // G], V[lo:end, h // G], Q[r, h]
                    x = k @ q * self.scale
                    e = (hd + 4) * self.scale * (np.abs(k) @ np.abs(q)).max()
                    if self.cap:
                        e += 8 * self.cap if largest >= 0.69 * self.cap else 16 * np.abs(x).max()
                        x = self.cap * np.tanh(x / self.cap)
                    if self.slopes is not None:
                        b = float(self.slopes[h]) * ago
                        x = x - b
                        near = x > x.max() - 100                       # what weighs anything
                        e += 2 * b[near].max() + 6 * np.abs(x[near]).max()
                    else:
                        e += 6 * np.abs(x).max()
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    O[r, h] = w @ v
                    t = (u + 2 * e * 2.0 ** -24 + 1.5 * n * 2.0 ** -24) * (w @ np.abs(v))
                    tol[r, h] = t + u * (np.abs(O[r, h]) + t) + 2.0 ** -24
        return O.reshape(self.n_rows, -1), tol.reshape(self.n_rows, -1)


def documents(P, M, starts, percent=0):
    """Spans of the rows of a sequence of documents that start at `starts`, the first `percent` of each seen whichever way round."""
    q = P + np.arange(M)
    starts = np.asarray(starts)
    ends = np.append(starts[1:], P + M)
    at = np.searchsorted(starts, q, side="right") - 1
    return np.stack([starts[at], starts[at] + (ends[at] - starts[at]) * percent // 100], -1)
