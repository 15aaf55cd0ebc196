"""A decode step made of the operators that stand around the differential attention, as a chain on the device:
adapters on the projection -> attn_prep with its append -> attn_diff -> logits and history -> chain_advance, the chosen token's row
of a table being the next step's hidden row. Every step's parts against their own references, a captured chain against the eager one."""
import numpy as np
import pytest
import torch

import test_gpu_logits as logits
import test_gpu_lowrank as lowrank
from diff_utils import HD, DiffCase
from espetero_amd import abi, device, host, synth
from test_gpu_diff import check, dev

pytestmark = pytest.mark.gpu

K = 5
P0 = [70, 33, 15, 0]
H, HKV, BT, D, RANK = 8, 4, 16, 256, 16
V = H * HD                                                            # the attention's output row is taken for the logits
SLICES = [(0, H * HD), (H * HD, HKV * HD), (H * HD + HKV * HD, HKV * HD)]


@pytest.mark.parametrize("dtype", [abi.ESP_F16, abi.ESP_BF16])
def test_a_chain_of_steps(dtype):
    device.init(0)
    n, tdt = len(P0), logits.TORCH[dtype]
    rng = np.random.default_rng(5)
    full = DiffCase(H, HKV, dtype, BT, [(P + K, 1) for P in P0], seed=1)
    full.scale = 1.0                                                  # the prep scales the queries
    full.trees["P"] = P0
    full.seqs = [(P, 1) for P in P0]
    ap = full.params()
    resident, groups = device.attn_diff_hint(ap)
    tiles, jobs, parts = host.plan_tiles(full.trees, groups, 0, None, host.options_mi355x(ap.rows_per_tile, resident))
    d = device.diff_params(dev(full.weight), dev(full.norm_w), full.eps, full.factor)
    dp = device.DiffPass(ap, d, full.trees, host.open_ended(tiles, full.trees), jobs, parts, n, full.block_list, pool_blocks=full.n_blocks)
    pp, a = synth.make_prep("omni", H, HKV, HD, dtype, n, seed=2, bt=BT)
    lr = lowrank.Case([0, 2, -1, 1], D, RANK, SLICES, dtype, 3, seed=3, y_ld=pp.x_ld)
    lp = device.LowRankPass(device.lowrank_params(D, RANK, SLICES, dtype, D, pp.x_ld, 3), lr.adapter)
    lg = logits.Case(n, V, dtype, seed=4)
    gp = device.LogitsPass(device.logits_params(V, dtype, lg.n_slots, len(lg.allowed), len(lg.bias_tokens)), lg.rows, lg.bias_tokens)

    base = dev(rng.standard_normal((K, n, pp.x_ld)).astype(np.float32))
    table = dev(synth._bits(rng.standard_normal((V, D)).astype(np.float32), dtype)).view(tdt)
    pos0, rows0 = np.zeros((n, 4), np.int32), np.full((n, 4), -1, np.int32)
    pos0[:, :3] = np.array(P0)[:, None]
    rows0[:, 0], rows0[:, 1] = full.block_list[full.trees["table"] + np.array(P0) // BT], np.array(P0) % BT
    init = dict(trees=device.to_dev(full.trees), pos=dev(pos0), rows=dev(rows0), pool=dev(full.pool), hidden=dev(lr.X).view(tdt),
                seen=dev(logits.words(np.stack([lg.prompt, lg.counts > 0], 1))), counts=dev(lg.counts), X=base)
    st = {k: v.clone() for k, v in init.items()}
    dp.trees = st["trees"]
    A, B, scale, blocks = dev(lr.A), dev(lr.B), dev(lr.scale), dev(full.block_list)
    prep = [dev(a[k]) if a[k] is not None else None for k in ("qn_w", "kn_w", "inv_freq", "rope_sel")]
    bt, bv, masks = dev(lg.bias_tokens), dev(lg.bias_values), dev(logits.words(lg.allowed))
    out = dict(hidden=torch.zeros(K, n, D, dtype=tdt, device="cuda"), Q=torch.zeros(K, n, H * HD, dtype=torch.int16, device="cuda"),
               O=torch.zeros(K, n, H * HD, dtype=torch.int16, device="cuda"), logits=torch.zeros(K, n, V, device="cuda"),
               tokens=torch.zeros(K, n, dtype=torch.int32, device="cuda"))

    def chain():
        for s in range(K):
            out["hidden"][s].copy_(st["hidden"])
            lp.run(st["hidden"], A, B, scale, st["X"][s])
            device.attn_prep(pp, st["X"][s], prep[0], prep[1], st["pos"], prep[2], prep[3], out["Q"][s], None, None, st["rows"], st["pool"], n)
            dp.run(out["Q"][s], st["pool"], out["O"][s])
            gp.run(out["O"][s], out["logits"][s], out["tokens"][s], bt, bv, masks, st["seen"], st["counts"], record=True)
            torch.index_select(table, 0, out["tokens"][s], out=st["hidden"])
            device.chain_advance(st["trees"], n, st["pos"], st["rows"], blocks, BT)

    def reset():
        for k, v in init.items():
            st[k].copy_(v)
        for t in out.values():
            t.zero_()

    chain()
    torch.cuda.synchronize()
    eager = {k: v.cpu().clone() for k, v in {**st, **out}.items()}
    u16 = lambda t: t.view(torch.int16).numpy().view(np.uint16)  # noqa: E731
    # The caches as the chain left them, token by token.
    full.K, full.V = [], []
    for i, P in enumerate(P0):
        k, v = (torch.zeros(P + K, HKV * HD, dtype=torch.int16, device="cuda") for _ in range(2))
        device.kv_gather(ap, st["pool"], blocks[int(full.trees["table"][i]):], P + K, k, v)
        torch.cuda.synchronize()
        full.K.append(k.cpu().numpy().view(np.uint16).reshape(-1, HKV, HD))
        full.V.append(v.cpu().numpy().view(np.uint16).reshape(-1, HKV, HD))
    for s in range(K):
        lr.X, lr.Y = u16(eager["hidden"][s]), base[s].cpu().numpy()
        want, tol = lr.expected()
        assert np.all(np.abs(eager["X"][s].numpy() - want) <= tol), s
        full.seqs, full.Q = [(P + s, 1) for P in P0], u16(eager["Q"][s])
        check(full, u16(eager["O"][s]))
        lg.L = eager["O"][s].view(tdt)
        want, tokens = lg.expected()
        assert np.array_equal(eager["logits"][s].numpy(), want) and (eager["tokens"][s].numpy() == tokens).all(), s
        for r, t in zip(lg.rows, tokens):
            lg.counts[r["slot"], t] += 1
        if s + 1 < K:
            assert torch.equal(eager["hidden"][s + 1].view(torch.int16), table.cpu()[torch.from_numpy(tokens).long()].view(torch.int16))
    assert (eager["counts"].numpy() == lg.counts).all()
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
        for k, v in {**st, **out}.items():
            assert torch.equal(v.cpu().view(torch.uint8), eager[k].view(torch.uint8)), (rep, k)
