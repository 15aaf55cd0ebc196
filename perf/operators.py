"""Three operators of a serving step around the paged-KV attention, timed in their plain form and as the library's kernels:

  diff      differential attention over the paged cache: the difference of two softmax maps of a pair of query heads over one
            pair of KV heads, with a learned weight per pair, a norm over the pair's output and a factor. The pass's rows are in
            the pool already. `seqs` sequences of `rows` rows each (`rows_lo` .. `rows` where prompts differ in length) behind
            `lo` .. `hi` cached keys, drawn from `lens`.
  lowrank   the low-rank adapters of many requests beside the fused projection in front of the attention: every row adds its
            own adapter's product to the fp32 projection, in place. `adapters` of them over `reqs` requests of `rows_lo` .. `rows`
            rows; the projection has the column slices `w0`, `w1`, `w2`, `gap` columns of something else between them.
  logits    the end of a decode step: penalties for repeated tokens, biases and a grammar's mask on the logits of `rows` requests,
            the best token of each, and its entry in the request's history.
"""
import math
import random

import numpy as np
import torch

own = False

F16, BF16, F32 = "fp16", "bf16", "fp32"
_TORCH = {F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32}
_HD = 128           # dims of a head; a pair's output has twice as many


def _diff(heads, dtype, bt, **kw):
    return dict(dict(op="diff", H=heads[0], Hkv=heads[1], dtype=dtype, bt=bt, window=0, seqs=1, lo=0, hi=0, rows_lo=0, rows=1, lens=1), **kw)


def _lowrank(widths, dtype, D, rank, **kw):
    return dict(dict(op="lowrank", w0=widths[0], w1=widths[1], w2=widths[2], dtype=dtype, D=D, rank=rank, gap=0, adapters=1, reqs=1, rows_lo=1,
                     rows=1, lens=1), **kw)


def _logits(vocab, dtype, rows, **kw):
    return dict(dict(op="logits", vocab=vocab, dtype=dtype, rows=rows, seen=500, bias=0, masks=0, keep=True, lens=1), **kw)


def listed():
    named = lambda name, c: dict(c, name=name)  # noqa: E731
    return [
        # One user, a short conversation: the smallest call, launches and latency.
        named("diff_one", _diff((16, 4), F16, 16, lo=1000, hi=1000)),
        # Two dozen users, contexts from a prompt to a long conversation: the everyday decode batch.
        named("diff_batch", _diff((32, 8), BF16, 16, seqs=24, lo=300, hi=9000, lens=2)),
        # Few very long documents: the stream of the cache is everything.
        named("diff_long", _diff((32, 4), F16, 64, seqs=4, lo=50000, hi=60000, lens=3)),
        # Speculative decoding: four rows per sequence, each sees the ones in front of it.
        named("diff_drafts", _diff((32, 8), BF16, 16, seqs=6, lo=2000, hi=16000, rows=4, lens=4)),
        # A handful of fresh user prompts of ragged lengths in one pass.
        named("diff_prompts", _diff((32, 8), F16, 16, seqs=5, rows_lo=40, rows=800, lens=5)),
        # A 2048-row chunk near the end of a long document: the largest product.
        named("diff_chunk", _diff((40, 8), BF16, 16, lo=12000, hi=12000, rows=2048)),
        # One request with a small adapter: the smallest call.
        named("lowrank_one", _lowrank((2048, 256, 256), F16, 2048, 8)),
        # A decode batch of many tenants: 48 requests over 20 adapters.
        named("lowrank_decode", _lowrank((5120, 1024, 1024), BF16, 5120, 16, adapters=20, reqs=48, lens=2)),
        # Prompt chunks of three tenants beside each other: the projection read and written once.
        named("lowrank_prompts", _lowrank((4096, 1024, 1024), BF16, 4096, 64, adapters=3, reqs=5, rows_lo=200, rows=700, lens=3)),
        # One request, a small vocabulary.
        named("logits_one", _logits(32000, F32, 1)),
        # A decode batch with an odd vocabulary, biases and grammars on half of the requests, 16-bit logits.
        named("logits_batch", _logits(50257, BF16, 48, seen=2000, bias=100, masks=3, lens=2)),
        # A full server on a large vocabulary, long histories; nobody reads the logits again, only the tokens count.
        named("logits_full", _logits(250000, F32, 192, seen=6000, bias=300, masks=8, keep=False, lens=3)),
    ]


_PAIRS = [(32, 8), (32, 4), (16, 4), (40, 8), (16, 8), (8, 2), (8, 8), (12, 4)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    what = rng.choice(["decode", "decode", "drafts", "prompts", "chunk", "sliding", "few", "many", "rows", "logits", "logits"])
    dtype, lens = rng.choice([F16, BF16]), rng.randrange(1 << 20)
    bt, pair = rng.choice([16, 16, 32, 64]), rng.choice(_PAIRS)
    if what == "decode":
        hi = _log(rng, 100, 60000)
        return _diff(pair, dtype, bt, seqs=_log(rng, 1, 64), lo=max(1, hi // rng.choice([1, 4, 16])), hi=hi, lens=lens)
    if what == "drafts":
        hi = _log(rng, 100, 20000)
        return _diff(pair, dtype, bt, seqs=_log(rng, 1, 16), lo=max(1, hi // rng.choice([1, 8])), hi=hi, rows=rng.randint(2, 8), lens=lens)
    if what == "prompts":
        hi = _log(rng, 20, 2000)
        return _diff(pair, dtype, bt, seqs=_log(rng, 1, 8), rows_lo=max(1, hi // rng.choice([1, 4, 16])), rows=hi, lens=lens)
    if what == "chunk":
        P = _log(rng, 10, 14000)
        return _diff(pair, dtype, bt, lo=P, hi=P, rows=_log(rng, 60, 2048), lens=lens)
    if what == "sliding":
        hi, rows = _log(rng, 200, 8000), rng.choice([1, 1, _log(rng, 30, 800)])
        return _diff(pair, dtype, bt, seqs=rng.randint(1, 6), lo=max(1, hi // rng.choice([1, 4])), hi=hi, rows_lo=max(1, rows // 2), rows=rows,
                     window=rng.choice([100, 512, 1000]), lens=lens)
    if what == "logits":
        bias = rng.choice([0, _log(rng, 1, 300)])
        return _logits(rng.choice([32000, 50257, 100003, 128256, 200064, 250000]), rng.choice([F32, F16, BF16]), _log(rng, 1, 192), seen=_log(rng, 1, 8000),
                       bias=bias, masks=rng.choice([0, rng.randint(1, 8)]), keep=rng.random() < 0.5, lens=lens)
    widths = rng.choice([(4096, 1024, 1024), (5120, 1024, 1024), (2048, 256, 256), (2560, 640, 640), (1536, 256, 1000)])
    D, rank, gap = rng.choice([1024, 2048, 2560, 4096, 5120]), rng.choice([8, 16, 24, 32, 64, 128]), rng.choice([0, 0, 128])
    if what == "few":
        return _lowrank(widths, dtype, D, rank, gap=gap, adapters=rng.randint(1, 4), reqs=_log(rng, 1, 8), lens=lens)
    if what == "many":
        return _lowrank(widths, dtype, D, min(rank, 32), gap=gap, adapters=_log(rng, 2, 30), reqs=_log(rng, 4, 128), lens=lens)
    rows = _log(rng, 10, 1500)
    return _lowrank(widths, dtype, D, rank, gap=gap, adapters=rng.randint(1, 4), reqs=rng.randint(1, 6), rows_lo=max(1, rows // rng.choice([1, 4])), rows=rows,
                    lens=lens)


def draw(rng):
    """One more case of these ranges, no larger than the largest listed one and within what the plain form has memory for."""
    most = max(_cost(c) for c in listed())
    while True:
        c = _drawn(rng)
        if _cost(c) <= most and _padded(c) <= 1.2e9:
            return c


def _cost(case):
    w = work(case)
    return w["flops"] / 8e14 + w["bytes"] / 4e12


def _padded(case):
    """Elements of the plain form's largest intermediate."""
    if case["op"] != "diff":
        return 0
    L = case["hi"] + case["rows"]
    return case["seqs"] * L * max(case["rows"] * case["H"], 4 * case["Hkv"] * _HD)


def _sequences(case):
    """[(cached keys, rows)] of the pass."""
    rng = random.Random(case["lens"])
    return [(rng.randint(case["lo"], case["hi"]), rng.randint(case["rows_lo"] or case["rows"], case["rows"])) for _ in range(case["seqs"])]


def _requests(case):
    """[(adapter, rows)] of the requests; an adapter of -1 is a request without one (the first has one)."""
    rng = random.Random(case["lens"])
    return [(rng.randrange(-1 if i else 0, case["adapters"]), rng.randint(case["rows_lo"], case["rows"])) for i in range(case["reqs"])]


def _bias_masks(case):
    """(entries of the bias list, row of the mask table) of every request."""
    rng = random.Random(case["lens"])
    return [(rng.choice([0, case["bias"]]), rng.choice([-1, rng.randrange(case["masks"])]) if case["masks"] else -1) for _ in range(case["rows"])]


def work(case):
    if case["op"] == "diff":
        pairs = keys = rows = 0
        for P, M in _sequences(case):
            q = P + np.arange(M, dtype=np.int64)
            pairs += int((np.minimum(q + 1, case["window"]) if case["window"] else q + 1).sum())
            keys += M + (min(P, case["window"] - 1) if case["window"] else P)
            rows += M
        return {"bytes": 2 * _HD * (2 * rows * case["H"] + 2 * keys * case["Hkv"]),    # Q in, O out; every visible key and value
                "flops": 6 * _HD * case["H"] * pairs}                                   # per head: 2 x 128 scores, 2 x 256 of P V
    if case["op"] == "lowrank":
        reqs, out = _requests(case), case["w0"] + case["w1"] + case["w2"]
        rows = sum(n for a, n in reqs if a >= 0)
        used = len({a for a, _ in reqs if a >= 0})
        per_row = 2 * case["D"] + 2 * 4 * out
        return {"bytes": rows * per_row + used * 2 * case["rank"] * (3 * case["D"] + out),
                "flops": 2 * rows * case["rank"] * (3 * case["D"] + out)}
    e = 4 if case["dtype"] == F32 else 2
    n = case["rows"] * case["vocab"]
    words = 4 * ((case["vocab"] + 31) // 32)
    masked = sum(m >= 0 for _, m in _bias_masks(case))
    return {"bytes": n * (e + (4 if case["keep"] else 0)) + case["rows"] * (2 * words + 4 * min(case["seen"], case["vocab"])) + masked * words, "flops": 0}


# ---- inputs -------------------------------------------------------------------------------------------------------------

class _State:
    pass


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = _State()
    s.case = dict(case)
    {"diff": _prepare_diff, "lowrank": _prepare_lowrank, "logits": _prepare_logits}[case["op"]](s, case, gen)
    return s


def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _prepare_diff(s, case, gen):
    H, Hkv, bt, tdt = case["H"], case["Hkv"], case["bt"], _TORCH[case["dtype"]]
    seqs = _sequences(case)
    n_rows = sum(M for _, M in seqs)
    per = [-(-(P + M) // bt) for P, M in seqs]
    n_blocks = sum(per)
    # The pool in the library's layout: per block and KV head, K [bt][128], then V in groups of 16 tokens, [bt / 16][128][16].
    s.pool = _normal(gen, n_blocks * 2 * bt * Hkv * _HD, tdt)
    s.pool.view(n_blocks * Hkv, 2, bt * _HD)[:, 1] *= 0.5
    s.blocks = torch.randperm(n_blocks, generator=gen, device="cuda").to(torch.int32)
    s.Q = _normal(gen, (n_rows, H * _HD), tdt)
    s.O = torch.zeros_like(s.Q)
    s.weight = torch.empty(H // 2, dtype=torch.float32, device="cuda").uniform_(0.2, 0.8, generator=gen)
    s.norm_w = _normal(gen, 2 * _HD, torch.float32, 0.1, 1.0)
    s.scale, s.eps, s.factor = _HD ** -0.5, 1e-5, 0.7
    s.P, s.M = np.array([P for P, _ in seqs]), np.array([M for _, M in seqs])
    s.base, s.table = np.cumsum(s.M) - s.M, np.cumsum(per) - np.array(per)
    # Where the rows and pages of every sequence lie, padded to the longest.
    last, pages = np.arange(s.M.max()), np.arange(max(per))
    s.row_of = _dev(s.base[:, None] + np.minimum(last, s.M[:, None] - 1))
    s.page_of = _dev(s.table[:, None] + np.minimum(pages, np.array(per)[:, None] - 1))
    s.qpos = _dev(s.P[:, None] + np.minimum(last, s.M[:, None] - 1))
    s.real = _dev((last < s.M[:, None]).reshape(-1).nonzero()[0])
    if own:
        from espetero_amd import abi, device, host, synth
        device.init(0)
        rows = int(s.M.max())
        p = synth.make_params(H, Hkv, _HD, abi.ESP_F16 if case["dtype"] == F16 else abi.ESP_BF16, bt, window=case["window"], scale=s.scale,
                              rows_per_tile=rows)
        p.rows_per_tile = device.attn_diff_rows(p, rows)
        d = device.diff_params(s.weight, s.norm_w, s.eps, s.factor)
        trees, pos = np.zeros(len(seqs), abi.TREE_DT), np.zeros((n_rows, 4), np.int32)
        for i, (P, M) in enumerate(seqs):
            trees[i] = (s.base[i], P, s.table[i], M)
            pos[s.base[i]:s.base[i] + M, :3] = (P + np.arange(M))[:, None]
        resident, groups = device.attn_diff_hint(p)
        tiles, jobs, n_parts = host.plan_tiles(trees, groups, case["window"], pos if case["window"] else None,
                                               host.options_mi355x(p.rows_per_tile, resident))
        s.dp = device.DiffPass(p, d, trees, tiles, jobs, n_parts, n_rows, s.blocks.cpu().numpy(), pool_blocks=n_blocks)


def _prepare_lowrank(s, case, gen):
    tdt, D, r, na = _TORCH[case["dtype"]], case["D"], case["rank"], case["adapters"]
    widths = [case["w0"], case["w1"], case["w2"]]
    reqs = _requests(case)
    s.adapter = np.concatenate([np.full(n, a, np.int32) for a, n in reqs])
    n_rows = len(s.adapter)
    s.off = [case["gap"], 2 * case["gap"] + widths[0], 3 * case["gap"] + widths[0] + widths[1]]
    s.y_ld = s.off[2] + widths[2]
    s.X = _normal(gen, (n_rows, D), tdt)
    s.Y = _normal(gen, (n_rows, s.y_ld), torch.float32)
    s.A = _normal(gen, (na, 3 * r, D), tdt, D ** -0.5)                       # every slice's rows of A, one under the other
    s.B = _normal(gen, (na, sum(widths), r), tdt, 0.5 * r ** -0.5)           # and of B
    s.factor = torch.empty(na, dtype=torch.float32, device="cuda").uniform_(0.5, 2.0, generator=gen)
    s.which = _dev(s.adapter.astype(np.int64))
    if own:
        from espetero_amd import abi, device
        device.init(0)
        p = device.lowrank_params(D, r, list(zip(s.off, widths)), abi.ESP_F16 if case["dtype"] == F16 else abi.ESP_BF16, D, s.y_ld, na)
        s.lp = device.LowRankPass(p, s.adapter)


def _prepare_logits(s, case, gen):
    rows, V = case["rows"], case["vocab"]
    s.W = (V + 31) // 32
    s.L = _normal(gen, (rows, V), torch.float32, 3.0).to(_TORCH[case["dtype"]])
    slots = 2 * rows
    s.slot = torch.randperm(slots, generator=gen, device="cuda")[:rows]
    # Histories: a prompt's tokens and those that were given out since, few of them often.
    n = case["seen"]
    prompt = torch.randint(V, (slots, n), generator=gen, device="cuda")
    given = (V * torch.rand((slots, n), generator=gen, device="cuda") ** 3).long().clamp_(max=V - 1)
    s.counts = torch.zeros(slots, V, dtype=torch.int32, device="cuda")
    s.counts.scatter_add_(1, given, torch.ones_like(given, dtype=torch.int32))
    was = torch.zeros(slots, 2, s.W * 32, dtype=torch.bool, device="cuda")
    was[:, 0].scatter_(1, prompt, True)
    was[:, 1, :V] = s.counts > 0
    s.seen = _words(was)
    per = _bias_masks(case)
    total = sum(b for b, _ in per)
    s.bias0 = np.cumsum([b for b, _ in per]) - np.array([b for b, _ in per])
    tokens = [torch.randperm(V, generator=gen, device="cuda")[:b].sort().values for b, _ in per if b]
    s.bias_tokens = torch.cat(tokens).to(torch.int32) if total else torch.zeros(1, dtype=torch.int32, device="cuda")
    s.bias_values = _normal(gen, max(total, 1), torch.float32, 5.0)
    s.bias_row = _dev(np.repeat(np.arange(rows), [b for b, _ in per]))
    s.n_bias = total
    allowed = torch.rand((max(case["masks"], 1), s.W * 32), generator=gen, device="cuda") < 0.3
    s.masks = _words(allowed)
    s.mask_row = _dev(np.array([m for _, m in per]))
    s.repetition = torch.empty(rows, device="cuda").uniform_(1.0, 1.3, generator=gen)
    s.frequency = torch.empty(rows, device="cuda").uniform_(0.0, 0.5, generator=gen)
    s.presence = torch.empty(rows, device="cuda").uniform_(0.0, 0.5, generator=gen)
    s.out = torch.empty(rows, V, dtype=torch.float32, device="cuda") if case["keep"] else None
    s.tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    if own:
        from espetero_amd import abi, device
        device.init(0)
        dt = {F16: abi.ESP_F16, BF16: abi.ESP_BF16, F32: abi.ESP_F32}[case["dtype"]]
        p = device.logits_params(V, dt, slots, case["masks"], s.n_bias)
        rec = np.zeros(rows, abi.LOGITS_ROW_DT)
        rec["slot"], rec["mask"] = s.slot.cpu().numpy(), [m for _, m in per]
        rec["bias0"], rec["n_bias"] = s.bias0, [b for b, _ in per]
        rec["repetition"], rec["frequency"], rec["presence"] = (x.cpu().numpy() for x in (s.repetition, s.frequency, s.presence))
        s.lp = device.LogitsPass(p, rec)


def _words(bits):
    """Truth values [..., 32 W] as 32-bit words [..., W], the first in the lowest bit."""
    b = bits.view(*bits.shape[:-1], -1, 32).to(torch.int64) << torch.arange(32, device="cuda")
    w = b.sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _bits(words, V):
    return ((words.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1).flatten(-2)[..., :V].bool()


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(s):
    op = s.case["op"]
    if own:
        if op == "diff":
            s.dp.run(s.Q, s.pool, s.O)
            return s.O
        if op == "lowrank":
            s.lp.run(s.X, s.A, s.B, s.factor, s.Y)
            return s.Y
        s.lp.run(s.L, s.out, s.tokens, s.bias_tokens, s.bias_values, s.masks, s.seen, s.counts, record=True)
    else:
        if op == "diff":
            s.O = _plain_diff(s)
            return s.O
        if op == "lowrank":
            return _plain_lowrank(s)
        _plain_logits(s)
    return {"out": s.out, "tokens": s.tokens, "seen": s.seen, "counts": s.counts}


def _plain_diff(s):
    c, d = s.case, _HD
    H, Hkv, bt = c["H"], c["Hkv"], c["bt"]
    S, R = s.row_of.shape
    Np, G = Hkv // 2, H // Hkv
    page = s.pool.view(-1, Hkv, 2, bt * d)[s.blocks.long()[s.page_of]]                              # [S][pages][Hkv][2][bt d]
    L = page.shape[1] * bt
    K = page[:, :, :, 0].reshape(S, -1, Hkv, bt, d).permute(0, 2, 1, 3, 4).reshape(S, Np, 2, L, d).float()
    V = page[:, :, :, 1].reshape(S, -1, Np, 2, bt // 16, d, 16).permute(0, 2, 1, 4, 6, 3, 5).reshape(S, Np, L, 2 * d).float()
    Q = s.Q[s.row_of].view(S, R, Np, G, 2, d).permute(0, 2, 4, 3, 1, 5).reshape(S, Np, 2, G * R, d).float()
    scores = torch.matmul(Q, K.transpose(-1, -2).contiguous()).view(S, Np, 2, G, R, L)
    scores *= s.scale
    ago = s.qpos[:, :, None] - torch.arange(L, device="cuda")                                        # [S][R][L]
    hidden = (ago < 0) | (ago >= c["window"]) if c["window"] else ago < 0
    scores.masked_fill_(hidden[:, None, None, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    scores /= scores.sum(-1, keepdim=True)
    maps = scores[:, :, 0] - s.weight.view(1, Np, G, 1, 1) * scores[:, :, 1]
    out = torch.matmul(maps.view(S, Np, G * R, L), V).view(S, Np, G, R, 2 * d)
    out = out * torch.rsqrt(out.square().mean(-1, keepdim=True) + s.eps) * s.norm_w * s.factor
    return out.permute(0, 3, 1, 2, 4).reshape(S * R, H * d)[s.real].to(s.Q.dtype)


def _plain_lowrank(s):
    r, na = s.case["rank"], s.case["adapters"]
    mine = (s.which[:, None] == torch.arange(na, device="cuda")).float() * s.factor                  # [rows][adapters]
    low = (s.X.float() @ s.A.float().view(na * 3 * r, -1).t()).view(-1, na, 3, r) * mine[:, :, None, None]
    B = s.B.float()
    w0, w1, w2 = s.case["w0"], s.case["w1"], s.case["w2"]
    s.Y[:, s.off[0]:s.off[0] + w0] += low[:, :, 0].reshape(-1, na * r) @ B[:, :w0].transpose(1, 2).reshape(na * r, -1)
    s.Y[:, s.off[1]:s.off[1] + w1] += low[:, :, 1].reshape(-1, na * r) @ B[:, w0:w0 + w1].transpose(1, 2).reshape(na * r, -1)
    s.Y[:, s.off[2]:s.off[2] + w2] += low[:, :, 2].reshape(-1, na * r) @ B[:, w0 + w1:].transpose(1, 2).reshape(na * r, -1)
    return s.Y


def _plain_logits(s):
    V, slot = s.case["vocab"], s.slot
    x = s.L.float()
    seen = _bits(s.seen[slot], V)                                                                    # [rows][2][vocab]
    x = torch.where(seen[:, 0] | seen[:, 1], torch.where(x > 0, x / s.repetition[:, None], x * s.repetition[:, None]), x)
    n = s.counts[slot].float()
    x = x - s.frequency[:, None] * n - s.presence[:, None] * seen[:, 1].float()
    if s.n_bias:
        x[s.bias_row, s.bias_tokens.long()] += s.bias_values
    if s.case["masks"]:
        allowed = _bits(s.masks, V)[s.mask_row.clamp(min=0)] | (s.mask_row < 0)[:, None]
        x.masked_fill_(~allowed, float("-inf"))
    best = x.amax(-1, keepdim=True)
    token = torch.where(x == best, torch.arange(V, device="cuda"), V).amin(-1)
    if s.out is not None:
        s.out.copy_(x)
    s.tokens.copy_(token)
    s.counts[slot, token] += 1
    word = s.seen[slot, 1, token // 32]
    s.seen[slot, 1, token // 32] = word | (torch.ones_like(word) << (token % 32).int())


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"diff": _exact_diff, "lowrank": _exact_lowrank, "logits": _exact_logits}[case["op"]](s)


def _exact_diff(s):
    c, d = s.case, _HD
    H, Hkv, bt = c["H"], c["Hkv"], c["bt"]
    out = torch.zeros(s.Q.shape, dtype=torch.float64, device="cuda")
    pool = s.pool.view(-1, Hkv, 2, bt * d)
    for base, P, table, M in zip(s.base.tolist(), s.P.tolist(), s.table.tolist(), s.M.tolist()):
        n = P + M
        pages = pool[s.blocks[table:table + -(-n // bt)].long()]
        age = (P + torch.arange(M, device="cuda"))[:, None] - torch.arange(n, device="cuda")[None]
        seen = age >= 0
        if c["window"]:
            seen &= age < c["window"]
        for pair in range(H // 2):
            kv = 2 * (pair // (H // Hkv))
            v = torch.cat([pages[:, kv + e, 1].reshape(-1, d, 16).transpose(1, 2).reshape(-1, d)[:n] for e in (0, 1)], 1).double()
            maps = []
            for e in (0, 1):
                q = s.Q[base:base + M, (2 * pair + e) * d:(2 * pair + e + 1) * d].double()
                k = pages[:, kv + e, 0].reshape(-1, d)[:n].double()
                maps.append(torch.softmax((q @ k.t() * s.scale).masked_fill(~seen, -math.inf), -1))
            o = (maps[0] - float(s.weight[pair]) * maps[1]) @ v
            o = o / (o.pow(2).mean(1, keepdim=True) + s.eps).sqrt() * s.norm_w.double() * s.factor
            out[base:base + M, 2 * pair * d:2 * (pair + 1) * d] = o
    return out


def _exact_lowrank(s):
    out, r = s.Y.double(), s.case["rank"]
    widths = [s.case["w0"], s.case["w1"], s.case["w2"]]
    for a in range(s.case["adapters"]):
        rows = (s.which == a).nonzero()[:, 0]
        x, at = s.X[rows].double(), 0
        for i, (off, w) in enumerate(zip(s.off, widths)):
            add = x @ s.A[a, i * r:(i + 1) * r].double().t() @ s.B[a, at:at + w].double().t()
            out[rows[:, None], off + torch.arange(w, device="cuda")] += float(s.factor[a]) * add
            at += w
    return out


def _exact_logits(s):
    """The logits alone: which token is best hangs on the last bit where two are nearly alike."""
    if s.out is None:
        return None
    V, out = s.case["vocab"], []
    for i in range(s.case["rows"]):
        slot = int(s.slot[i])
        x, n = s.L[i].double(), s.counts[slot].double()
        known = (n > 0) | _bits(s.seen[slot, 0], V)
        rep = float(s.repetition[i])
        x = torch.where(known & (x > 0), x / rep, torch.where(known, x * rep, x))
        x = x - float(s.frequency[i]) * n - float(s.presence[i]) * (n > 0)
        mine = (s.bias_row == i).nonzero()[:, 0]
        x[s.bias_tokens[mine].long()] += s.bias_values[mine].double()
        m = int(s.mask_row[i])
        if m >= 0:
            x[~_bits(s.masks[m], V)] = -math.inf
        out.append(x)
    return {"out": torch.stack(out), "tokens": None, "seen": None, "counts": None}
