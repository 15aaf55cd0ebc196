"""esp_linear_attn on the device against the recurrence in float64."""
import ctypes as C

import numpy as np
import pytest
import torch

from linear_utils import LinearCase
from espetero_amd import abi, device
from oracle import binding as ob

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16
MARK = 0x1234


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16 if a.dtype == np.uint16 else a.dtype)).cuda()


class Run:
    def __init__(self, case, workgroups=None):
        device.init(0)
        self.case = case
        self.lp = device.LinearPass(case.params(), case.records, case.n_rows, workgroups=workgroups)
        self.Q, self.K, self.V, self.decay = dev(case.Q), dev(case.K), dev(case.V), dev(case.decay)
        self.states = dev(case.states) if case.n_states else None
        self.O = torch.full((case.n_rows, case.H * case.dv + case.wide), MARK, dtype=torch.int16, device="cuda")
        print(f"linear H{case.H}/{case.Hk} {case.dk}x{case.dv} dtype{case.dtype} seqs{case.seqs[:6]} tiles{self.lp.n_tiles} few{self.lp.n_few} "
              f"parts{self.lp.n_parts}", flush=True)

    def enqueue(self, stream=None):
        self.lp.run(self.Q, self.K, self.V, self.decay, self.states, self.O, stream=stream)

    def reset(self):
        self.O.fill_(MARK)
        if self.states is not None:
            self.states.copy_(dev(self.case.states))

    def __call__(self):
        self.enqueue()
        torch.cuda.synchronize()
        return self.out()

    def out(self):
        return self.O.cpu().numpy().view(np.uint16).copy(), None if self.states is None else self.states.cpu().numpy().copy()


def check(case, got):
    bits, states = got
    want, tol, S, tolS = case.expected()
    w = case.H * case.dv
    live = np.isfinite(want[:, 0])
    o = ob.to_f32(bits[:, :w], case.dtype).astype(np.float64)
    worst = np.max(np.abs(o[live] - want[live]) / tol[live]) if live.any() else 0.0
    off = np.abs(states - S) if states is not None else np.zeros(1)
    worst_s = np.max(off / np.maximum(tolS, 1e-300)) if states is not None and off.size else 0.0
    print(f"  of the bound: O {worst:.3f} states {worst_s:.3f}", flush=True)
    assert np.all(np.abs(o[live] - want[live]) <= tol[live]), worst
    assert (bits[~live] == MARK).all() and (bits[:, w:] == MARK).all()
    if states is not None:
        assert np.all(off <= tolS), worst_s                          # slots that nobody leaves a state in: bit for bit


DIMS = [(64, 64), (64, 128), (128, 64), (128, 128), (128, 256), (64, 192), (128, 512)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dk,dv", DIMS)
@pytest.mark.parametrize("row_decay", [False, True])
def test_single_tokens_and_drafts(dk, dv, dtype, row_decay):
    c = LinearCase(4, 2, dk, dv, dtype, [(1, 0, 0), (1, -1, 1), (5, 2, 3), (16, 4, -1), (2, 4, 5), (0, 4, 6), (0, -1, 7), (0, 8, 8), (1, -1, -1)],
                   n_states=10, row_decay=row_decay, seed=dk + dv)
    check(c, Run(c)())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dk,dv", DIMS)
@pytest.mark.parametrize("row_decay", [False, True])
def test_prompts(dk, dv, dtype, row_decay):
    c = LinearCase(2, 1, dk, dv, dtype, [(17, 0, 0), (64, -1, 1), (65, 2, 3), (200, 2, -1), (127, 4, 5), (3, 6, 6)], n_states=8, row_decay=row_decay,
                   seed=dk + dv)
    check(c, Run(c, workgroups=1)())
    check(c, Run(c, workgroups=4096)())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("to", ["same", "fork", "fresh", "nowhere"])
def test_segments_of_a_long_sequence(to, dtype):
    src, dst = {"same": (1, 1), "fork": (1, 0), "fresh": (-1, 0), "nowhere": (1, -1)}[to]
    c = LinearCase(3, 3, 128, 128, dtype, [(900, src, dst)], n_states=2, seed=3)
    r = Run(c, workgroups=4096)
    assert r.lp.n_parts > 3
    check(c, r())


@pytest.mark.parametrize("heads", [(1, 1), (5, 5), (6, 2), (16, 1), (40, 8)])
def test_heads(heads):
    c = LinearCase(*heads, 64, 64, BF16, [(33, 0, 0), (1, 1, 1), (130, -1, 2)], seed=heads[0])
    check(c, Run(c)())


def test_many_sequences_fill_wide_workgroups():
    c = LinearCase(8, 8, 128, 128, BF16, [(1, i, i) for i in range(140)], seed=4)
    check(c, Run(c)())
    c = LinearCase(8, 4, 64, 64, F16, [(1 + i % 3, i, 140 + i) for i in range(140)], n_states=280, seed=5, row_decay=True)
    check(c, Run(c)())


@pytest.mark.parametrize("decay", [0.0, -1e-4, -3.0, -60.0, -200.0, float("-inf"), 1.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decays(decay, dtype):
    c = LinearCase(2, 2, 64, 64, dtype, [(150, 0, 0), (4, 1, 1)], seed=6, decay=decay)
    check(c, Run(c, workgroups=1)())
    check(c, Run(c, workgroups=4096)())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_row_that_forgets_everything(dtype):
    """Log decays of minus infinity at some rows: what lies in front of them is gone, and what lies between them keeps its bits."""
    c = LinearCase(2, 2, 64, 64, dtype, [(300, 0, 0), (9, 1, 1)], seed=7, row_decay=True)
    c.decay[[0, 40, 41, 63, 64, 130, 303]] = -np.inf
    c.decay[100:128] = -100.0
    c.decay[200:230] = 0.0
    check(c, Run(c, workgroups=1)())
    check(c, Run(c, workgroups=4096)())


@pytest.mark.parametrize("std", [1e-3, 30.0, 2000.0])
def test_sizes_of_fp16_numbers(std):
    c = LinearCase(2, 2, 128, 128, F16, [(180, 0, 0), (5, 1, 1)], seed=8, size=std, scale=128 ** -0.5 / std ** 2)
    c.states *= np.float32(std * std)
    check(c, Run(c)())


def test_the_last_of_a_lone_token_in_an_fp16_chunk():
    """One token, then 63 of zeros under a strong decay: the state is that token's, far below the values it was made from."""
    for dtype in (F16, BF16):
        c = LinearCase(1, 1, 64, 64, dtype, [(64, -1, 0), (100, -1, 1)], seed=9, decay=-1.2)
        c.V[1:64] = 0
        c.K[70:] = 0
        check(c, Run(c, workgroups=1)())


def test_columns_of_very_different_sizes():
    for dtype in (F16, BF16):
        c = LinearCase(1, 1, 128, 128, dtype, [(130, 0, 0)], seed=10)
        V = ob.to_f32(c.V, dtype)
        V[:, ::2] *= 2.0 ** -12
        c.V = ob.from_f32(V.reshape(-1), dtype).reshape(c.V.shape)
        c.states[..., ::2] *= np.float32(2.0 ** -12)
        bits, states = Run(c)()
        want, _, S, tolS = c.expected()
        err = np.abs(ob.to_f32(bits, dtype)[:, ::2] - want[:, ::2])
        assert err.max() <= (2.0 ** -11 if dtype == F16 else 2.0 ** -8) * 1.2 * np.abs(want[:, ::2]).max()
        assert (np.abs(states - S) <= tolS).all()


def test_strides_and_rows_of_nobody():
    c = LinearCase(4, 2, 64, 128, BF16, [(70, 0, 0), (2, 1, 1)], n_states=4, seed=11, gap=7, wide=24)
    check(c, Run(c)())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [9, 120, 500])
@pytest.mark.parametrize("what", ["Q", "K", "V"])
def test_what_is_not_finite_stays_behind_its_row(what, rows, dtype):
    c = LinearCase(2, 2, 64, 64, dtype, [(rows, 0, 0), (rows, 1, 1)], seed=12)
    workgroups = 4096 if rows == 500 else 1
    clean, _ = Run(c, workgroups)()
    r0 = rows * 3 // 5
    inf = 0x7C00 if dtype == F16 else 0x7F80
    for bad in (inf, inf | 0x8000, inf | 1):
        x = getattr(c, what).copy()
        getattr(c, what)[r0, 5] = bad
        bits, states = Run(c, workgroups)()
        setattr(c, what, x)
        assert (bits[:r0] == clean[:r0]).all(), (what, bad)
        assert (bits[rows:] == clean[rows:]).all()                   # the other sequence
        assert (bits[:, 64:] == clean[:, 64:]).all()                 # and the other head
        row = ob.to_f32(bits[r0, :64], dtype)
        assert not np.isfinite(row[5] if what == "V" else row).any()
        if what == "V":
            rest = np.arange(64) != 5
            assert np.isfinite(ob.to_f32(bits[:rows, :64], dtype)[:, rest]).all()
            assert not np.isfinite(states[0, 0, :, 5]).any() and np.isfinite(states[0, 0][:, rest]).all()
        if what == "Q":
            assert (bits[r0 + 1:rows] == clean[r0 + 1:rows]).all()


def test_an_infinite_state_shows_in_its_column_only():
    for dtype in (F16, BF16):
        c = LinearCase(1, 1, 64, 64, dtype, [(100, 0, 0)], seed=13)
        clean, _ = Run(c)()
        c.states[0, 0, 9, 5] = np.inf
        bits, states = Run(c)()
        rest = np.arange(64) != 5
        assert not np.isfinite(ob.to_f32(bits[:, 5], dtype)).any() and not np.isfinite(states[0, 0, 9, 5])
        assert np.isfinite(states[0, 0][:, rest]).all()
        assert (bits[:, rest] == clean[:, rest]).all()


def test_a_chunk_at_a_time_is_the_whole():
    """A prompt in chunks of odd lengths, then single tokens, through one slot: as the recurrence of all of it."""
    whole = LinearCase(4, 4, 128, 64, BF16, [(333, -1, 0)], seed=14)
    want, tol, S, tolS = whole.expected()
    r = Run(whole)
    at, first = 0, True
    for rows in (100, 17, 64, 130, 1, 1, 4, 16):
        seqs = np.zeros(1, abi.LINEAR_SEQ_DT)
        seqs[0] = (at, rows, -1 if first else 0, 0)
        first = False
        r.lp = device.LinearPass(whole.params(), seqs, whole.n_rows)
        r.enqueue()
        at += rows
    assert at == 333
    torch.cuda.synchronize()
    bits, states = r.out()
    o = ob.to_f32(bits, BF16)
    assert (np.abs(o - want) <= 1.1 * tol).all() and (np.abs(states - S) <= 2 * tolS).all()   # eight sets of roundings instead of six chunks'


def test_another_stream_a_second_pass_and_a_graph_give_the_same_bits():
    c = LinearCase(4, 4, 128, 128, F16, [(700, 0, 0), (1, 1, 1), (90, -1, 2), (4, 1, 3)][:3], n_states=4, seed=15)
    r = Run(c, workgroups=2048)
    assert r.lp.n_parts > 0
    bits, states = r()
    r.reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    r.enqueue(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    b2, s2 = r.out()
    assert (b2 == bits).all() and (s2 == states).all()
    g = torch.cuda.CUDAGraph()
    r.reset()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        r.enqueue()
    for _ in range(3):
        r.reset()
        g.replay()
        torch.cuda.synchronize()
        b2, s2 = r.out()
        assert (b2 == bits).all() and (s2 == states).all()
    # Replays go on from the states that the one in front has left.
    r.reset()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    by_graph = r.out()
    r.reset()
    for _ in range(3):
        r.enqueue()
    torch.cuda.synchronize()
    again = r.out()
    assert (by_graph[0] == again[0]).all() and (by_graph[1] == again[1]).all()


def test_two_graphs_with_a_workspace_each():
    runs = [Run(LinearCase(2, 2, 128, 128, BF16, [(600, 0, 0)], seed=s), workgroups=4096) for s in (16, 17)]
    eager = [r() for r in runs]
    graphs = []
    for r in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r.enqueue()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for r in runs:
            r.reset()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for r, e in zip(runs, eager):
            b, s = r.out()
            assert (b == e[0]).all() and (s == e[1]).all()


def test_states_past_32_bit_offsets():
    """A slot whose state starts behind the first 2^31 numbers."""
    c = LinearCase(64, 64, 128, 256, BF16, [(1, 0, 1), (70, 2, 2)], n_states=3, seed=18)
    slot = 64 * 128 * 256
    far = (1 << 31) // slot + 3
    r = Run(c)
    want = r()
    check(c, want)
    big = torch.empty((far + 3) * slot, dtype=torch.float32, device="cuda")
    big[far * slot:].copy_(dev(c.states).view(-1))
    moved = LinearCase(64, 64, 128, 256, BF16, [(1, 0, 1), (70, 2, 2)], n_states=3, seed=18)
    p = moved.params()
    p.n_states = far + 3
    seqs = moved.records.copy()
    seqs["src"] += far
    seqs["dst"] += far
    r.lp = device.LinearPass(p, seqs, c.n_rows)
    r.states = big
    r.O.fill_(MARK)
    r.enqueue()
    torch.cuda.synchronize()
    assert (r.O.cpu().numpy().view(np.uint16) == want[0]).all()
    assert (big[far * slot:].cpu().numpy().reshape(c.states.shape) == want[1]).all()
    del big


def test_the_workspace_is_checked():
    c = LinearCase(2, 2, 128, 128, F16, [(900, 0, 0)], seed=19)
    r = Run(c, workgroups=4096)
    need = abi.attn_lib().esp_linear_workspace_bytes(C.byref(r.lp.params), r.lp.n_parts)
    r.lp.workspace = torch.empty(need - 1, dtype=torch.uint8, device="cuda")
    with pytest.raises(abi.EspError, match="workspace"):
        r()
