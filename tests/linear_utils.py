"""Linear attention for the tests: small cases, the operator in float64, and how far a kernel that rounds as the library says may be
from it."""
import numpy as np

from espetero_amd import abi, device, host, synth
from oracle import binding as ob

HALF = {abi.ESP_F16: 2.0 ** -11, abi.ESP_BF16: 2.0 ** -8}     # half a step of the storage type, relative


class LinearCase:
    """seqs: (rows, src slot, dst slot). Rows of the sequences follow each other behind `gap` rows that are nobody's; columns behind the
    heads and those rows hold NaN. decay: log decays of a head, drawn over the heads and, with row_decay, over the rows too."""

    def __init__(self, H, Hk, dk, dv, dtype, seqs, n_states=None, row_decay=False, seed=0, gap=0, wide=0, decay=None, scale=None, size=1.0):
        rng = np.random.default_rng(seed)
        self.H, self.Hk, self.dk, self.dv, self.dtype, self.seqs, self.row_decay = H, Hk, dk, dv, dtype, list(seqs), row_decay
        self.n_states = n_states if n_states is not None else max([0] + [max(s, d) + 1 for _, s, d in seqs])
        self.n_rows = gap + sum(r for r, _, _ in seqs)
        self.scale = dk ** -0.5 if scale is None else scale
        nan = np.uint16(0x7E00 if dtype == abi.ESP_F16 else 0x7FC0)

        def rows(heads, d, std):
            x = np.full((self.n_rows, heads * d + wide), nan, np.uint16)
            x[gap:, :heads * d] = synth._bits(rng.standard_normal((self.n_rows - gap, heads * d), dtype=np.float32) * np.float32(std), dtype)
            return x
        self.Q, self.K, self.V = rows(Hk, dk, size), rows(Hk, dk, dk ** -0.5), rows(H, dv, size)
        self.wide = wide
        self.states = rng.standard_normal((self.n_states, H, dk, dv)).astype(np.float32)
        d = -np.exp2(-8.0 * (1 + np.arange(H)) / H) if decay is None else np.full(H, decay)
        if row_decay:
            d = d * np.exp(rng.standard_normal((self.n_rows, H)))
        self.decay = d.astype(np.float32)
        self.records = np.zeros(len(seqs), abi.LINEAR_SEQ_DT)
        base = gap
        for i, (r, s, t) in enumerate(seqs):
            self.records[i] = (base, r, s, t)
            base += r

    def params(self):
        H, Hk, dk, dv, w = self.H, self.Hk, self.dk, self.dv, self.wide
        return device.linear_params(H, Hk, dk, dv, self.dtype, self.scale, self.n_states, row_decay=self.row_decay, q_ld=Hk * dk + w,
                                    k_ld=Hk * dk + w, v_ld=H * dv + w, o_ld=H * dv + w)

    def plan(self, workgroups=512):
        return host.plan_linear(self.params(), self.records, self.n_rows, workgroups)

    def expected(self):
        """O [n_rows][H * dv] (NaN where no sequence has a row), states, and how far the kernel's may be from them, in float64.

        Of the terms of a sum: a weight exp(c) is off by the fp32 exponential's own step and by c's, |c| 2^-24 log2 units, and what is
        |c| > 150 weighs nothing: 2^-16.5 at most, |c| taken as 150. P and S enter products as two numbers of the storage type: 2^-16
        (bf16) at most each. The sums themselves are fp32: a product over dk, one over dk and 64 rows, 3 operations a chunk on the
        state. So O may be off by t A, A the sum of the terms' sizes, and by its rounding. A state's terms enter as numbers of 22 bits or
        more; their weights are off by the exponentials of as many chunks. Behind those, the 2^-38 of the largest that fp16 scales lose, and
        what fp32 cannot hold of a state: 2^-126 for each of the 64 terms of a chunk and the operations on it."""
        H, Hk, dk, dv = self.H, self.Hk, self.dk, self.dv
        f = lambda x, heads, d: ob.to_f32(x[:, :heads * d], self.dtype).astype(np.float64).reshape(-1, heads, d)  # noqa: E731
        Q, K = (np.repeat(f(x, Hk, dk), H // Hk, 1) for x in (self.Q, self.K))
        V = f(self.V, H, dv)
        O = np.full((self.n_rows, H, dv), np.nan)
        tolO = np.full_like(O, np.nan)
        states, tolS = self.states.astype(np.float64), np.zeros(self.states.shape)
        u, old = HALF[self.dtype], states.copy()
        for base, rows, src, dst in self.records.tolist():
            S = old[src].copy() if src >= 0 else np.zeros((H, dk, dv))
            A, at, big = np.abs(S), 0.0, 0.0
            for r in range(base, base + rows):
                d = np.minimum(self.decay[r] if self.row_decay else self.decay, 0).astype(np.float64)
                lam = np.where(d < -138, 0.0, np.exp(np.maximum(d, -138)))[:, None, None]
                kv = K[r][:, :, None] * V[r][:, None, :]
                S, A = lam * S + kv, lam * A + np.abs(kv)
                O[r] = self.scale * np.einsum("hk,hkv->hv", Q[r], S)
                n_chunks = 1 + (r - base) // 64
                t = 2.0 ** -14.5 + (2 * dk + 64 + 6 * n_chunks) * 2.0 ** -24
                big = max(big, A.max())
                a = abs(self.scale) * (np.einsum("hk,hkv->hv", np.abs(Q[r]), A) + 2.0 ** -38 * big * np.abs(Q[r]).sum(-1)[:, None])
                tolO[r] = t * a + u * (np.abs(O[r]) + t * a) + (2.0 ** -25 if self.dtype == abi.ESP_F16 else 0)
                at = max(at, -float(d.min()) * 1.45 * (r - base + 1))
            if dst >= 0:
                states[dst] = S
                chunks = (rows + 63) // 64
                tolS[dst] = (16 + 64 + 8 * chunks + min(at, 150.0)) * 2.0 ** -24 * A + 2.0 ** -38 * A.max((1, 2), keepdims=True) \
                    + 80 * chunks * 2.0 ** -126 if rows else 0.0
        return O.reshape(self.n_rows, H * dv), tolO.reshape(self.n_rows, H * dv), states, tolS
