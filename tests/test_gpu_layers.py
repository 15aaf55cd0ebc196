"""Layers of two kinds in turn over the same sequences, as a hybrid decoder runs them: linear attention on slices of one row of numbers
-> its output on top of a projection -> attn_prep with its append -> attention with shaped scores, whose output is the next step's row. First the
prompts (sequences of packed documents, a prefix), then a chain of single tokens with chain_advance between them, eager and captured. Every part
against its own reference."""
import copy

import numpy as np
import pytest
import torch

from espetero_amd import abi, device, host, synth
from linear_utils import LinearCase
from shaped_utils import ShapedCase, documents
import test_gpu_linear as linear
import test_gpu_shaped as shaped
from test_gpu_shaped import dev

pytestmark = pytest.mark.gpu

K = 4
P0 = [70, 130, 1, 33]
H, HKV, HD, BT = 8, 2, 128, 16
LH, LK, DK, DV = 4, 2, 64, 128                                        # its rows: [q 2 x 64][k 2 x 64][v 4 x 128] of 1024 numbers
WIDTH = H * HD
Q_AT, K_AT, V_AT = 0, LK * DK, 2 * LK * DK
DOCS = [[0, 40], [0], [0], [0, 5, 20]]
PREFIX = [25, 60, 0, 40]                                              # percent of a document


def rows_of(case, rows, u):
    """case, a LinearCase, on the rows u [n][WIDTH] of storage bits."""
    case.n_rows, case.records = sum(rows), np.zeros(len(rows), abi.LINEAR_SEQ_DT)
    case.Q, case.K, case.V = u[:, Q_AT:], u[:, K_AT:], u[:, V_AT:]
    case.records["base"] = np.cumsum([0] + rows)[:-1]
    case.records["rows"] = rows
    return case


@pytest.mark.parametrize("cap,window", [(20.0, 0), (0.0, 0), (30.0, 48)])
@pytest.mark.parametrize("dtype", [abi.ESP_F16, abi.ESP_BF16])
def test_prompts_and_a_chain_of_steps(dtype, cap, window):
    device.init(0)
    n, n_pre = len(P0), sum(P0)
    u16 = lambda t: t.cpu().view(torch.int16).numpy().view(np.uint16)  # noqa: E731
    rng = np.random.default_rng(7)

    # The attention layer: K tokens of room behind the prompts.
    whole = [documents(0, P + K, d, c) for P, d, c in zip(P0, DOCS, PREFIX)]
    step = ShapedCase(H, HKV, HD, dtype, BT, [(P + K, 1) for P in P0], window=window, cap=cap, bias=True, seed=1)
    step.trees["P"], step.seqs = P0, [(P, 1) for P in P0]
    step.spans = np.array([(w[P][0], min(w[P][1], P)) for w, P in zip(whole, P0)], np.int32)   # (nobody sees a token that is not there yet)
    step.scale = 1.0                                                  # the prep scales the queries
    pre = copy.copy(step)
    pre.n_rows, pre.seqs, pre.trees = n_pre, [(0, M) for M in P0], step.trees.copy()
    pre.trees["P"], pre.trees["M"], pre.trees["base"] = 0, P0, np.cumsum([0] + P0)[:-1]
    pre.spans = np.concatenate([np.minimum(w[:P], P) for w, P in zip(whole, P0)]).astype(np.int32)
    pre.pos = np.zeros((n_pre, 4), np.int32)
    pre.pos[:, :3] = np.concatenate([np.arange(P) for P in P0])[:, None]
    step.pos = np.zeros((n, 4), np.int32)
    step.pos[:, :3] = np.array(P0)[:, None]

    def passes(case, open_ended):
        p = case.params()
        tiles, jobs, parts = case.plan(p)
        sp = device.ShapedPass(p, device.shape_params(cap, dev(case.slopes)), case.trees, host.open_ended(tiles, case.trees) if open_ended else tiles, jobs, parts,
                               case.n_rows, case.block_list, spans=case.spans, pool_blocks=case.n_blocks)
        lin = LinearCase(LH, LK, DK, DV, dtype, [(1, i, i) for i in range(n)], seed=2)
        lp = device.linear_params(LH, LK, DK, DV, dtype, DK ** -0.5, n, q_ld=WIDTH, k_ld=WIDTH, v_ld=WIDTH)
        rows = [M for _, M in case.seqs]
        rows_of(lin, rows, np.zeros((sum(rows), WIDTH), np.uint16))
        lin.records["src"], lin.records["dst"] = -1 if not open_ended else np.arange(n), np.arange(n)
        return sp, lin, device.LinearPass(lp, lin.records, case.n_rows)

    pre_sp, pre_lin, pre_lp = passes(pre, False)
    sp, lin, lp = passes(step, True)
    pp, a = synth.make_prep("omni", H, HKV, HD, dtype, n_pre, seed=3, bt=BT)
    prep = [dev(a[k]) if a[k] is not None else None for k in ("qn_w", "kn_w", "inv_freq", "rope_sel")]
    table = lambda case, pos: np.stack([step.block_list[case + pos // BT], pos % BT], -1).astype(np.int32)  # noqa: E731
    pre_rows, rows0 = np.full((n_pre, 4), -1, np.int32), np.full((n, 4), -1, np.int32)
    pre_rows[:, :2] = table(np.repeat(step.trees["table"], P0), pre.pos[:, 0])
    rows0[:, :2] = table(step.trees["table"], np.array(P0))
    first = dev(synth._bits(rng.standard_normal((n_pre, WIDTH)).astype(np.float32), dtype))
    base = dev(rng.standard_normal((K, n, pp.x_ld)).astype(np.float32))
    blocks, decay = dev(step.block_list), dev(lin.decay)
    tdt = torch.float16 if dtype == abi.ESP_F16 else torch.bfloat16

    def layers(hidden, lpass, states, X, pos, row_table, spass, pool, o1, q, o2, rows):
        lpass.run(hidden[:, Q_AT:], hidden[:, K_AT:], hidden[:, V_AT:], decay, states, o1)
        X[:, :LH * DV] += o1.view(tdt).float()
        device.attn_prep(pp, X, prep[0], prep[1], pos, prep[2], prep[3], q, None, None, row_table, pool, rows)
        spass.run(q, pool, o2)

    def out(*shape):
        return torch.zeros(*shape, dtype=torch.int16, device="cuda")

    # ---- the prompts
    pool, states = dev(step.pool), torch.full((n, LH, DK, DV), float("nan"), device="cuda")
    o1, q, o2, X = out(n_pre, LH * DV), out(n_pre, WIDTH), out(n_pre, WIDTH), dev(a["X"])
    layers(first, pre_lp, states, X, dev(pre.pos), dev(pre_rows), pre_sp, pool, o1, q, o2, n_pre)
    torch.cuda.synchronize()

    def cached(case, pool, lens):
        """The caches' first tokens as they are in the pool."""
        case.K, case.V = [], []
        p = case.params()
        for i, L in enumerate(lens):
            k, v = out(L, HKV * HD), out(L, HKV * HD)
            device.kv_gather(p, pool, blocks[int(step.trees["table"][i]):], L, k, v)
            torch.cuda.synchronize()
            case.K.append(u16(k).reshape(-1, HKV, HD))
            case.V.append(u16(v).reshape(-1, HKV, HD))

    cached(pre, pool, P0)
    rows_of(pre_lin, P0, u16(first))
    pre_lin.records["src"], pre_lin.records["dst"] = -1, np.arange(n)
    linear.check(pre_lin, (u16(o1), states.cpu().numpy()))
    pre.Q = u16(q)
    shaped.check(pre, u16(o2))

    # ---- single tokens
    last = torch.from_numpy(np.cumsum(P0) - 1).cuda()
    init = dict(trees=device.to_dev(step.trees), pos=dev(step.pos), rows=dev(rows0), pool=pool, states=states, X=base)
    st = {k: v.clone() for k, v in init.items()}
    sp.trees = st["trees"]
    got = dict(hidden=out(K + 1, n, WIDTH), o1=out(K, n, LH * DV), q=out(K, n, WIDTH), states=torch.zeros(K + 1, *states.shape, device="cuda"))
    start = o2[last].clone()

    def chain():
        got["hidden"][0].copy_(start)
        got["states"][0].copy_(st["states"])
        for s in range(K):
            layers(got["hidden"][s], lp, st["states"], st["X"][s], st["pos"], st["rows"], sp, st["pool"], got["o1"][s], got["q"][s], got["hidden"][s + 1], n)
            got["states"][s + 1].copy_(st["states"])
            device.chain_advance(st["trees"], n, st["pos"], st["rows"], blocks, BT)

    def reset():
        for k, v in init.items():
            st[k].copy_(v)
        for t in got.values():
            t.zero_()

    chain()
    torch.cuda.synchronize()
    eager = {k: v.cpu().clone() for k, v in {**st, **{"got " + k: v for k, v in got.items()}}.items()}
    cached(step, st["pool"], [P + K for P in P0])
    for s in range(K):
        rows_of(lin, [1] * n, u16(eager["got hidden"][s]))
        lin.records["src"] = lin.records["dst"] = np.arange(n)
        lin.states = eager["got states"][s].numpy()
        linear.check(lin, (u16(eager["got o1"][s]), eager["got states"][s + 1].numpy()))
        step.trees["P"] = np.array(P0) + s
        step.seqs, step.Q = [(P + s, 1) for P in P0], u16(eager["got q"][s])
        shaped.check(step, u16(eager["got hidden"][s + 1]))
    assert (eager["trees"].numpy().view(abi.TREE_DT)["P"] == np.array(P0) + K).all()

    g = torch.cuda.CUDAGraph()
    reset()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        chain()
    for rep in range(3):
        reset()
        if rep == 1:                                                  # eager work on the same buffers between the replays
            chain()
            torch.cuda.synchronize()
            reset()
        g.replay()
        torch.cuda.synchronize()
        for k, v in {**st, **{"got " + k: v for k, v in got.items()}}.items():
            assert torch.equal(v.cpu().view(torch.uint8), eager[k].view(torch.uint8)), (rep, k)


def test_two_streams_at_once():
    """A pass of each operator on a stream of its own, several times over, with the results that they have alone."""
    lins = [linear.Run(LinearCase(4, 4, 128, 128, abi.ESP_BF16, [(300, 0, 1), (3, 2, 2), (1, -1, 3)], seed=s)) for s in (1, 2)]
    shs = [shaped.Run(ShapedCase(8, 2, 128, abi.ESP_BF16, 16, [(400, 40), (0, 90)], cap=20.0, bias=True, seed=s)) for s in (3, 4)]
    for r in lins:
        r.reset()
    alone = [r() for r in lins] + [r() for r in shs]
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(3):
        for r in lins:
            r.reset()
        for r in shs:
            r.O.fill_(shaped.MARK)
        torch.cuda.synchronize()
        for r, s in zip(lins + shs, streams):
            r.enqueue(stream=s)
        torch.cuda.synchronize()
        for r, want in zip(lins, alone):
            assert all((x == y).all() for x, y in zip(r.out(), want))
        for r, want in zip(shs, alone[2:]):
            assert (r.bits() == want).all()
