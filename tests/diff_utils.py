"""Differential attention for the tests: small paged cases in the library's pool layout, the operator in float64, and how far a
kernel that rounds as the library says may be from it."""
import numpy as np

from espetero_amd import abi, device, host, synth
from oracle import binding as ob

HD = 128
HALF = {abi.ESP_F16: 2.0 ** -11, abi.ESP_BF16: 2.0 ** -8}     # half a step of the storage type, relative


class DiffCase:
    """seqs: (cached keys, rows). Rows and cached keys lie in the pool; memory that holds no key is filled with NaN."""

    def __init__(self, H, Hkv, dtype, bt, seqs, window=0, ring=False, seed=0, q_ld=None, norm=True, sharp=1.0, base_gap=0):
        rng = np.random.default_rng(seed)
        self.H, self.Hkv, self.dtype, self.bt, self.seqs, self.window = H, Hkv, dtype, bt, list(seqs), window
        bits = lambda x: synth._bits(x, dtype)  # noqa: E731
        nan = np.uint16(0x7E00 if dtype == abi.ESP_F16 else 0x7FC0)
        most = max(M for _, M in seqs)
        self.ring = -(-(window + most) // bt) if ring else 0
        per = [self.ring or -(-(P + M) // bt) for P, M in seqs]
        self.n_blocks = sum(per) + 2
        order = rng.permutation(self.n_blocks).astype(np.int32)
        self.n_rows = base_gap + sum(M for _, M in seqs)
        self.q_ld = q_ld or H * HD
        self.Q = np.full((self.n_rows, self.q_ld), nan, np.uint16)
        self.Q[:, :H * HD] = bits(rng.standard_normal((self.n_rows, H * HD), dtype=np.float32) * sharp)
        self.trees = np.zeros(len(seqs), abi.TREE_DT)
        self.pos = np.zeros((self.n_rows, 4), np.int32)
        k_plane = np.full((self.n_blocks, Hkv, bt, HD), nan, np.uint16)
        v_plane = np.full((self.n_blocks, Hkv, bt, HD), nan, np.uint16)
        self.K, self.V, self.block_list = [], [], order
        base, used = base_gap, 0
        for i, ((P, M), nb) in enumerate(zip(seqs, per)):
            n = P + M
            K, V = (rng.standard_normal((n, Hkv, HD), dtype=np.float32) * s for s in (1.0, 0.5))
            K, V = bits(K), bits(V)
            self.K.append(K)
            self.V.append(V)
            self.trees[i] = (base, P, used, M)
            self.pos[base:base + M, :3] = (P + np.arange(M))[:, None]
            for j in range(max(0, n - self.ring * bt) if ring else 0, n):
                b = used + (j // bt) % self.ring if ring else order[used + j // bt]
                k_plane[b, :, j % bt], v_plane[b, :, j % bt] = K[j], V[j]
            base += M
            used += nb
        vt = v_plane.reshape(self.n_blocks, Hkv, bt // 16, 16, HD).transpose(0, 1, 2, 4, 3).reshape(self.n_blocks, Hkv, bt * HD)
        self.pool = np.concatenate([k_plane.reshape(self.n_blocks, Hkv, bt * HD), vt], -1).reshape(-1)
        self.weight = rng.uniform(0.2, 0.8, H // 2).astype(np.float32)
        self.norm_w = (1.0 + 0.1 * rng.standard_normal(2 * HD)).astype(np.float32) if norm else None
        self.eps, self.factor, self.scale = 1e-5, 0.7, HD ** -0.5

    def params(self, rows_per_tile=None):
        p = synth.make_params(self.H, self.Hkv, HD, self.dtype, self.bt, window=self.window, ring=self.ring, scale=self.scale, rows_per_tile=1)
        p.q_ld = self.q_ld
        p.rows_per_tile = rows_per_tile or device.attn_diff_rows(p, max(M for _, M in self.seqs))
        return p

    def plan(self, p, workgroups=None, cut_batch=False):
        resident, groups = device.attn_diff_hint(p) if workgroups is None else (workgroups, p.Hkv // 2)
        o = host.options_mi355x(p.rows_per_tile, resident)
        if cut_batch:
            o.cut_batch, o.min_chunk, o.min_span, o.item_steps, o.part_steps = 1, 32, 32, 1, 0
        return host.plan_tiles(self.trees, groups, self.window, self.pos if self.window else None, o)

    def expected(self, rows=None):
        """(O, how far from it an output may be) in float64 at the rows asked for, [n_rows][H * 128] with NaN elsewhere.

        A kernel's unnormalised weights are off by a factor of 1 + d, |d| <= u + 2 e: u half a step of the storage type (P is rounded
        to it for the product with V), e what a score's fp32 sum of 128 products and its exponential are off. Sums over n keys in
        fp32 add n 2^-24. With A[d] = sum p1 |v_d| + w sum p2 |v_d| the difference is off by at most t A[d], t = u + 2 e + n 2^-24
        (weights summed in fp32, half of that again); the norm divides by r and changes by r's own error, at most rms(t A) / r;
        the result is rounded once: u |O|."""
        G = self.H // self.Hkv
        u = HALF[self.dtype]
        f = lambda x: ob.to_f32(x, self.dtype).astype(np.float64)  # noqa: E731
        Q = f(self.Q)
        O = np.full((self.n_rows, self.H * HD), np.nan)
        tol = np.full_like(O, np.nan)
        for i, (P, M) in enumerate(self.seqs):
            K, V = f(self.K[i]), f(self.V[i])
            base = int(self.trees["base"][i])
            for m in range(M):
                if rows is not None and base + m not in rows:
                    continue
                n = P + m + 1
                lo = max(0, n - self.window) if self.window else 0
                for pair in range(self.H // 2):
                    kv = 2 * (pair // G)
                    v = np.concatenate([V[lo:n, kv], V[lo:n, kv + 1]], -1)
                    o, A, t = np.zeros(2 * HD), np.zeros(2 * HD), 0.0
                    for e in (0, 1):
                        q = Q[base + m, (2 * pair + e) * HD:(2 * pair + e + 1) * HD]
                        s = K[lo:n, kv + e] @ q * self.scale
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        c = 1.0 if e == 0 else -float(self.weight[pair])
                        o += c * (w @ v)
                        A += abs(c) * (w @ np.abs(v))
                        es = 2.0 ** -24 * (132 * self.scale * (np.abs(K[lo:n, kv + e]) @ np.abs(q)).max() + 4 * np.abs(s).max() + 8)
                        t = max(t, u + 2 * es + 1.5 * (n - lo) * 2.0 ** -24)
                    d = t * A
                    if self.norm_w is not None:
                        r = np.sqrt((o * o).mean() + self.eps)
                        g = self.factor * self.norm_w.astype(np.float64) / r
                        d = np.abs(g) * (d + np.abs(o) * np.sqrt((d * d).mean()) / r) * (1 + 2.0 ** -20)
                        o = o * g
                    else:
                        o, d = o * self.factor, d * self.factor
                    at = slice(2 * pair * HD, 2 * (pair + 1) * HD)
                    O[base + m, at] = o
                    tol[base + m, at] = d + u * (np.abs(o) + d) + 2.0 ** -24
        return O, tol
