"""esp_logits_process and the histories on the device, bit for bit against numpy's fp32 in the documented order."""
import numpy as np
import pytest
import torch

from espetero_amd import abi, device

pytestmark = pytest.mark.gpu

F16, BF16, F32 = abi.ESP_F16, abi.ESP_BF16, abi.ESP_F32
TORCH = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}


def words(bits):
    """Truth values [..., V] -> 32-bit words [..., ceil(V / 32)]."""
    V = bits.shape[-1]
    pad = np.zeros(bits.shape[:-1] + (-(-V // 32) * 32,), bool)
    pad[..., :V] = bits
    return np.packbits(pad, axis=-1, bitorder="little").view("<u4").view(np.int32)


class Case:
    def __init__(self, n, V, dtype, seed=0, n_slots=None, n_masks=2, bias=20, in_ld=None, out_ld=None, ties=False):
        rng = np.random.default_rng(seed)
        self.n, self.V, self.dtype = n, V, dtype
        self.n_slots = n + 2 if n_slots is None else n_slots
        self.in_ld, self.out_ld = in_ld or V, out_ld or V
        x = rng.standard_normal((n, self.in_ld)).astype(np.float32) * 3
        if ties:
            x = np.round(x)
        self.L = torch.from_numpy(x).to(TORCH[dtype])
        self.prompt = rng.random((self.n_slots, V)) < 0.1
        self.counts = np.where(rng.random((self.n_slots, V)) < 0.1, rng.integers(1, 9, (self.n_slots, V)), 0).astype(np.int32)
        self.allowed = rng.random((n_masks, V)) < 0.4
        self.rows = np.zeros(n, abi.LOGITS_ROW_DT)
        self.rows["slot"] = rng.permutation(self.n_slots)[:n] if self.n_slots >= n else -1
        self.rows["mask"] = rng.integers(-1, n_masks, n) if n_masks else -1
        toks, vals = [], []
        for i in range(n):
            b = int(rng.integers(0, min(bias, V) + 1))
            self.rows[i]["bias0"], self.rows[i]["n_bias"] = sum(map(len, toks)), b
            toks.append(np.sort(rng.permutation(V)[:b]))
            vals.append(rng.standard_normal(b).astype(np.float32) * 5)
        self.bias_tokens, self.bias_values = np.concatenate(toks).astype(np.int32), np.concatenate(vals).astype(np.float32)
        self.rows["repetition"] = rng.uniform(0.9, 1.4, n)
        self.rows["frequency"], self.rows["presence"] = rng.uniform(-0.2, 0.5, (2, n))

    def expected(self):
        out, tokens = [], []
        for i, r in enumerate(self.rows):
            x = self.L[i, :self.V].float().numpy().copy()
            if r["slot"] >= 0:
                given = self.counts[r["slot"]] > 0
                known = given | self.prompt[r["slot"]]
                x = np.where(known, np.where(x > 0, x / r["repetition"], x * r["repetition"]), x)
                pen = x - r["frequency"] * self.counts[r["slot"]].astype(np.float32)
                x = np.where(given, pen - r["presence"], x)
            mine = slice(r["bias0"], r["bias0"] + r["n_bias"])
            x[self.bias_tokens[mine]] += self.bias_values[mine]
            if r["mask"] >= 0:
                x[~self.allowed[r["mask"]]] = -np.inf
            out.append(x.astype(np.float32))
            ok = ~np.isnan(x) & (x > -np.inf)
            tokens.append(int(np.argmax(np.where(ok, x, -np.inf))) if ok.any() else -1)
        return np.stack(out), np.array(tokens, np.int32)

    def prepare(self):
        device.init(0)
        self.p = device.logits_params(self.V, self.dtype, self.n_slots, len(self.allowed), len(self.bias_tokens), self.in_ld, self.out_ld)
        self.lp = device.LogitsPass(self.p, self.rows, self.bias_tokens)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda() if a.size else None  # noqa: E731
        self.dL, self.bt, self.bv = self.L.cuda(), dev(self.bias_tokens), dev(self.bias_values)
        self.masks = dev(words(self.allowed))
        self.seen = dev(words(np.stack([self.prompt, self.counts > 0], 1)))
        self.dcounts = dev(self.counts)
        self.out = torch.full((self.n, self.out_ld), 7.5, device="cuda")
        self.tokens = torch.full((self.n,), -9, dtype=torch.int32, device="cuda")
        print(f"logits rows{self.n} vocab{self.V} dtype{self.dtype} slots{self.n_slots} masks{len(self.allowed)} bias{len(self.bias_tokens)}", flush=True)
        return self

    def run(self, out=True, tokens=True, record=False):
        self.lp.run(self.dL, self.out if out else None, self.tokens if tokens else None, self.bt, self.bv, self.masks, self.seen, self.dcounts, record)

    def check(self):
        want, tokens = self.expected()
        self.prepare().run(record=self.n_slots > 0)
        torch.cuda.synchronize()
        out = self.out.cpu().numpy()
        assert np.array_equal(out[:, :self.V], want, equal_nan=True)
        assert (out[:, self.V:] == 7.5).all()
        assert (self.tokens.cpu().numpy() == tokens).all()
        if self.n_slots:
            counts = self.counts.copy()
            for r, t in zip(self.rows, tokens):
                if r["slot"] >= 0 and t >= 0:
                    counts[r["slot"], t] += 1
            assert (self.dcounts.cpu().numpy() == counts).all()
            assert (self.seen.cpu().numpy() == words(np.stack([self.prompt, counts > 0], 1))).all()
        return tokens


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,V", [(1, 1), (1, 7), (3, 31), (2, 33), (5, 1000), (4, 2047), (4, 2049), (9, 5003), (2, 40009)])
def test_sizes(n, V, dtype):
    Case(n, V, dtype, seed=V).check()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_ties_go_to_the_lowest_token(dtype):
    for seed in range(4):
        c = Case(6, 9001, dtype, seed=seed, ties=True, n_masks=0, bias=0)
        c.rows["repetition"], c.rows["frequency"], c.rows["presence"] = 1, 0, 0
        c.check()


def test_strides_and_rows_without_anything():
    for dtype in (F16, F32):
        Case(3, 4099, dtype, seed=1, in_ld=4105, out_ld=4103).check()
        Case(3, 4099, dtype, seed=2, n_slots=0, n_masks=0, bias=0).check()


@pytest.mark.parametrize("seen", [0.004, 0.05, 0.3, 0.95])
def test_in_place_every_token_is_penalised_once(seen):
    """Lists of a few tokens a chunk up to all of them, in many workgroups: no wavefront takes what another has written for a logit."""
    c = Case(192, 20011, F32, seed=29, n_masks=1, bias=40)
    rng = np.random.default_rng(31)
    c.prompt = rng.random(c.prompt.shape) < seen
    c.counts[:] = np.where(rng.random(c.counts.shape) < seen / 4, 3, 0)
    c.rows["repetition"], c.rows["mask"] = 1.5, -1
    want, tokens = c.expected()
    c.prepare()
    for _ in range(5):
        c.out = c.L.cuda()
        c.dL = c.out
        c.run()
        torch.cuda.synchronize()
        assert np.array_equal(c.out.cpu().numpy(), want) and (c.tokens.cpu().numpy() == tokens).all()


def test_alone_in_place_and_only_tokens():
    c = Case(4, 3001, F32, seed=3)
    want, tokens = c.expected()
    c.prepare().run(tokens=False)
    torch.cuda.synchronize()
    assert np.array_equal(c.out.cpu().numpy(), want) and (c.tokens == -9).all()
    c.prepare().run(out=False)
    torch.cuda.synchronize()
    assert (c.tokens.cpu().numpy() == tokens).all() and (c.out == 7.5).all()
    c.prepare()
    c.out = c.dL
    c.run()
    torch.cuda.synchronize()
    assert np.array_equal(c.dL.cpu().numpy(), want) and (c.tokens.cpu().numpy() == tokens).all()


def test_nothing_left_infinities_and_nan():
    c = Case(6, 3000, F32, seed=4, bias=0)
    c.rows["repetition"], c.rows["frequency"], c.rows["presence"] = 1, 0, 0
    c.allowed[1] = False
    c.rows["mask"] = [-1, -1, 1, -1, 0, -1]
    c.L[0] = float("nan")
    c.L[1] = float("-inf")
    c.L[3, 2500] = float("nan")
    c.L[3, 17] = float("inf")
    c.L[4, ~torch.from_numpy(c.allowed[0])] = float("nan")
    c.L[5, 100:] = float("nan")
    tokens = c.check()
    assert list(tokens[:4]) == [-1, -1, -1, 17] and tokens[4] >= 0 and 0 <= tokens[5] < 100


def test_records_outside_their_arrays_count_as_none():
    c = Case(3, 500, F32, seed=5)
    c.rows["slot"], c.rows["mask"] = [-1, 10**6, -5], [-7, 5, 2]
    c.rows["bias0"], c.rows["n_bias"] = [10**6, -3, 2**31 - 1], [5, -1, 5]
    p = device.logits_params(c.V, c.dtype, c.n_slots, len(c.allowed), len(c.bias_tokens))
    device.init(0)
    lp = device.LogitsPass(p, c.rows)                                   # unchecked
    c.rows = c.rows.copy()
    c.rows["slot"], c.rows["mask"], c.rows["n_bias"], c.rows["bias0"] = -1, -1, 0, 0
    want, tokens = c.expected()
    c.prepare()
    c.lp = lp
    c.run(record=True)
    torch.cuda.synchronize()
    assert np.array_equal(c.out.cpu().numpy(), want) and (c.tokens.cpu().numpy() == tokens).all()
    assert (c.dcounts.cpu().numpy() == c.counts).all()


def test_rows_that_share_a_slot_record_together():
    c = Case(5, 2000, F32, seed=6, n_slots=1, bias=0, n_masks=0)
    c.rows["slot"] = 0
    c.rows["repetition"], c.rows["frequency"], c.rows["presence"] = 1, 0, 0
    c.L[:] = c.L[:1].clone()
    tokens = c.check()
    assert (tokens == tokens[0]).all()


def test_histories_are_recorded_and_cleared():
    c = Case(2, 1003, F32, seed=7, n_slots=4).prepare()
    device.history_clear(c.p, c.seen, c.dcounts, torch.tensor([1, 3, 1, 99, -1], dtype=torch.int32, device="cuda"), 5)
    torch.cuda.synchronize()
    prompt, counts = c.prompt.copy(), c.counts.copy()
    prompt[[1, 3]], counts[[1, 3]] = False, 0
    tokens = np.array([5, 5, 1002, 1003, -1, 40, 5, 0], np.int32)
    slots = np.array([1, 1, 1, 1, 1, 9, 3, -1], np.int32)
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    device.history_record(c.p, c.seen, c.dcounts, dev(tokens), dev(slots), len(tokens), True)
    device.history_record(c.p, c.seen, c.dcounts, dev(tokens[::-1].copy()), dev(slots[::-1].copy()), len(tokens), False)
    torch.cuda.synchronize()
    counts[1, 5] += 2
    counts[1, 1002] += 1
    counts[3, 5] += 1
    prompt[1, [5, 1002]] = prompt[3, 5] = True
    assert (c.dcounts.cpu().numpy() == counts).all()
    assert (c.seen.cpu().numpy() == words(np.stack([prompt, counts > 0], 1))).all()


def test_a_captured_step_goes_on_from_the_history_it_leaves():
    """Greedy steps on the same logits: what has been given out is penalised in the next replay, as in eager steps."""
    c = Case(3, 5000, BF16, seed=8)
    c.rows["frequency"] = 2.0
    c.prepare()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(record=True)
    for _ in range(4):
        want, tokens = c.expected()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(c.out.cpu().numpy(), want) and (c.tokens.cpu().numpy() == tokens).all()
        for r, t in zip(c.rows, tokens):
            c.counts[r["slot"], t] += 1
    assert (c.dcounts.cpu().numpy() == c.counts).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_a_pass_of_many_tokens(dtype):
    Case(97, 131001, dtype, seed=9, bias=300, in_ld=131003, out_ld=131002).check()


@pytest.mark.parametrize("share", [0.0, 0.5, 1.0])
def test_histories_from_empty_to_every_token(share):
    for dtype in (BF16, F32):
        c = Case(4, 4099, dtype, seed=10, bias=400)
        rng = np.random.default_rng(11)
        c.prompt = rng.random(c.prompt.shape) < share
        c.counts = np.where(rng.random(c.counts.shape) < share, c.counts + 1, 0).astype(np.int32)
        c.check()


def test_bits_behind_the_vocabulary_are_not_looked_at():
    c = Case(3, 1001, F32, seed=12)
    want, tokens = c.expected()
    c.prepare()
    for words_ in (c.seen.view(-1, c.seen.shape[-1]), c.masks):
        words_[:, -1] |= -(1 << (1001 % 32))
    c.run()
    torch.cuda.synchronize()
    assert np.array_equal(c.out.cpu().numpy(), want) and (c.tokens.cpu().numpy() == tokens).all()
