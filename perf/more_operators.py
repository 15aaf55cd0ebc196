"""Two kinds of attention layer of a serving step, timed in their plain form and as the library's kernels:

  linear    linear attention with a decay for each head: a state of dk x dv numbers in place of a cache. `seqs` sequences of `rows`
            rows each (`rows_lo` .. `rows` where they differ in length, drawn from `lens`) go on from the states in their slots and
            leave them there (`to`: "same"), in another slot each ("fork"), or start from nothing ("fresh"). `H` heads of values and
            states, `Hk` heads of queries and keys. `gated`: a log decay for every row and head, else one for every head.
  shaped    softmax attention over the paged cache with shaped scores: capped by a tanh (`cap`), with a bias that falls with the
            distance (`bias`), each row seeing the keys of its own document (`docs` of them in a sequence, 0: one that is the sequence)
            and those of the document's first `prefix` percent whole, whichever way round. `seqs` sequences of `rows_lo` .. `rows`
            rows behind `lo` .. `hi` cached keys, drawn from `lens`. The pass's rows are in the pool already.
"""
import math
import random

import numpy as np
import torch

own = False

F16, BF16 = "fp16", "bf16"
_TORCH = {F16: torch.float16, BF16: torch.bfloat16}
_CHUNK = 64         # rows that the plain form of linear attention takes at a time


def _linear(heads, dims, dtype, **kw):
    return dict(dict(op="linear", H=heads[0], Hk=heads[1], dk=dims[0], dv=dims[1], dtype=dtype, seqs=1, rows_lo=0, rows=1, to="same", gated=False,
                     lens=1), **kw)


def _shaped(heads, hd, dtype, bt, **kw):
    return dict(dict(op="shaped", H=heads[0], Hkv=heads[1], hd=hd, dtype=dtype, bt=bt, window=0, seqs=1, lo=0, hi=0, rows_lo=0, rows=1, cap=0.0,
                     bias=False, docs=0, prefix=0, lens=1), **kw)


def listed():
    named = lambda name, c: dict(c, name=name)  # noqa: E731
    return [
        # One user's next token: the smallest call, launches and latency.
        named("linear_one", _linear((16, 16), (128, 128), F16)),
        # A full decode batch: every state read and written once, the stream of the states is everything.
        named("linear_batch", _linear((32, 32), (128, 128), BF16, seqs=64)),
        # Speculative decoding: a few rows per sequence, the states after them in slots of their own until the drafts are accepted.
        named("linear_drafts", _linear((32, 16), (128, 128), BF16, seqs=12, rows_lo=3, rows=6, to="fork", gated=True, lens=2)),
        # A handful of fresh user prompts of ragged lengths in one pass.
        named("linear_prompts", _linear((32, 32), (128, 128), F16, seqs=5, rows_lo=40, rows=900, to="fresh", lens=3)),
        # A long document in one pass, small heads, a decay for every row.
        named("linear_long", _linear((32, 8), (64, 128), BF16, rows=16000, gated=True, lens=4)),
        # Chunks of prompts of several users who each fill the pass's budget of rows: the largest product.
        named("linear_chunks", _linear((40, 40), (128, 128), BF16, seqs=4, rows=2048, lens=5)),
        # One user, a short conversation, capped scores: the smallest call.
        named("shaped_one", _shaped((16, 4), 128, F16, 16, lo=1000, hi=1000, cap=50.0)),
        # Two dozen users, contexts from a prompt to a long conversation, biased by distance: the everyday decode batch.
        named("shaped_batch", _shaped((32, 8), 128, BF16, 16, seqs=24, lo=300, hi=9000, bias=True, lens=2)),
        # Drafts on heads of 256 dims with capped scores and a sliding window.
        named("shaped_drafts", _shaped((16, 8), 256, F16, 64, seqs=8, lo=2000, hi=12000, rows=4, cap=30.0, window=4000, lens=3)),
        # Packed prompts: several documents behind each other, none sees another.
        named("shaped_docs", _shaped((32, 8), 128, F16, 16, seqs=3, rows_lo=500, rows=2000, docs=6, bias=True, lens=4)),
        # Prompts that open with an image or an instruction that is seen whole, heads of 256 dims.
        named("shaped_prefix", _shaped((8, 4), 256, BF16, 16, seqs=4, rows_lo=200, rows=1200, cap=50.0, prefix=40, lens=5)),
        # A 2048-row chunk near the end of a long document, capped and biased: the largest product.
        named("shaped_chunk", _shaped((32, 8), 128, BF16, 16, lo=8000, hi=8000, rows=2048, cap=50.0, bias=True)),
    ]


_HEADS = [(32, 32), (16, 16), (40, 40), (32, 8), (8, 8), (20, 4), (16, 2), (5, 5)]
_PAIRS = {128: [(32, 8), (32, 4), (16, 4), (40, 8), (16, 8), (8, 2), (8, 8), (12, 4), (7, 1)], 256: [(8, 4), (16, 8), (16, 4), (8, 1), (4, 4), (10, 2)]}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    what = rng.choice(["tokens", "tokens", "verify", "prompts", "long", "decode", "decode", "drafts", "fresh", "fresh", "chunk", "packed"])
    dtype, lens = rng.choice([F16, BF16]), rng.randrange(1 << 20)
    heads, dims = rng.choice(_HEADS), rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (128, 64), (128, 256)])
    gated, to = rng.random() < 0.5, rng.choice(["same", "same", "fork", "fresh"])
    if what == "tokens":
        return _linear(heads, dims, dtype, seqs=_log(rng, 1, 100), to=to, gated=gated, lens=lens)
    if what == "verify":
        return _linear(heads, dims, dtype, seqs=_log(rng, 1, 32), rows_lo=1, rows=rng.randint(2, 12), to=to, gated=gated, lens=lens)
    if what == "prompts":
        rows = _log(rng, 13, 2000)
        return _linear(heads, dims, dtype, seqs=_log(rng, 1, 12), rows_lo=max(1, rows // rng.choice([1, 4, 16])), rows=rows, to=to, gated=gated, lens=lens)
    if what == "long":
        return _linear(heads, dims, dtype, rows=_log(rng, 1000, 16000), to=to, gated=gated, lens=lens)
    hd, bt = rng.choice([128, 128, 256]), rng.choice([16, 16, 32, 64])
    pair = rng.choice(_PAIRS[hd])
    shape = dict(cap=rng.choice([0.0, 20.0, 50.0]), bias=rng.random() < 0.5, window=rng.choice([0, 0, 0, _log(rng, 100, 4000)]), lens=lens)
    if what == "decode":
        hi = _log(rng, 100, 30000)
        return _shaped(pair, hd, dtype, bt, seqs=_log(rng, 1, 48), lo=max(1, hi // rng.choice([1, 4, 16])), hi=hi, docs=rng.choice([0, 0, 0, 4]), **shape)
    if what == "drafts":
        hi = _log(rng, 100, 16000)
        return _shaped(pair, hd, dtype, bt, seqs=_log(rng, 1, 16), lo=max(1, hi // rng.choice([1, 8])), hi=hi, rows=rng.randint(2, 8), **shape)
    if what == "chunk":
        P = _log(rng, 10, 10000)
        return _shaped(pair, hd, dtype, bt, lo=P, hi=P, rows=_log(rng, 60, 2048), docs=rng.choice([0, 3]), prefix=rng.choice([0, 0, 30]), **shape)
    rows = _log(rng, 20, 2000)
    docs = rng.randint(2, 10) if what == "packed" else 0
    return _shaped(pair, hd, dtype, bt, seqs=_log(rng, 1, 8), rows_lo=max(1, rows // rng.choice([1, 4, 16])), rows=rows, docs=docs,
                   prefix=rng.choice([0, 0, 25, 60]), **shape)


def draw(rng):
    """One more case of these ranges, no larger than the largest listed one and within what the plain form has memory for."""
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("linear", "shaped")}
    while True:
        c = _drawn(rng)
        if _cost(c) <= most[c["op"]] and _padded(c) <= 8e8:
            return c


def _cost(case):
    w = work(case)
    return w["flops"] / 8e14 + w["bytes"] / 4e12


def _padded(case):
    """Elements of the plain form's largest intermediate."""
    if case["op"] == "linear":
        return case["seqs"] * case["rows"] * case["H"] * (case["dk"] + case["dv"])
    L = case["hi"] + case["rows"]
    return case["seqs"] * L * max(case["rows"] * case["H"], 2 * case["Hkv"] * case["hd"])


def _rows(case):
    rng = random.Random(case["lens"])
    return [rng.randint(case["rows_lo"] or case["rows"], case["rows"]) for _ in range(case["seqs"])]


def _sequences(case):
    """[(cached keys, rows)] of the pass."""
    rng = random.Random(case["lens"])
    return [(rng.randint(case["lo"], case["hi"]), rng.randint(case["rows_lo"] or case["rows"], case["rows"])) for _ in range(case["seqs"])]


def _spans(case):
    """For every row of every sequence, the start of its document and the end of what it sees of it whichever way round."""
    rng, out = random.Random(case["lens"] + 1), []
    for P, M in _sequences(case):
        n = P + M
        starts = np.array([0] + sorted(rng.randrange(n) for _ in range(case["docs"] - 1)) if case["docs"] else [0])
        ends = np.append(starts[1:], n)
        which = np.searchsorted(starts, P + np.arange(M), side="right") - 1
        first = starts[which]
        out.append(np.stack([first, first + (ends[which] - first) * case["prefix"] // 100], -1))
    return out


def _visible(case):
    """[(first, end)] arrays over the rows of each sequence: the keys that a row sees."""
    out = []
    for (P, M), span in zip(_sequences(case), _spans(case)):
        q = P + np.arange(M)
        first = np.maximum(span[:, 0], q - case["window"] + 1) if case["window"] else span[:, 0]
        out.append((first, np.maximum(q + 1, span[:, 1])))
    return out


def work(case):
    if case["op"] == "linear":
        rows = sum(_rows(case))
        H, dk, dv = case["H"], case["dk"], case["dv"]
        states = case["seqs"] * (1 if case["to"] == "fresh" else 2)
        return {"bytes": 2 * rows * (2 * case["Hk"] * dk + 2 * H * dv) + 4 * H * dk * dv * states + 4 * H * (rows if case["gated"] else 1),
                "flops": 4 * rows * H * dk * dv}
    pairs = keys = rows = 0
    for first, end in _visible(case):
        pairs += int((end - first).sum())
        keys += _covered(first, end)
        rows += len(first)
    hd = case["hd"]
    return {"bytes": 2 * hd * (2 * rows * case["H"] + 2 * keys * case["Hkv"]),          # Q in, O out; every visible key and value
            "flops": 4 * hd * case["H"] * pairs}


def _covered(first, end):
    """Keys that some row sees."""
    mark = np.zeros(int(end.max()) + 1, np.int64)
    np.add.at(mark, first, 1)
    np.add.at(mark, end, -1)
    return int((np.cumsum(mark) > 0).sum())


# ---- inputs -------------------------------------------------------------------------------------------------------------

class _State:
    pass


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = _State()
    s.case = dict(case)
    {"linear": _prepare_linear, "shaped": _prepare_shaped}[case["op"]](s, case, gen)
    return s


def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _prepare_linear(s, case, gen):
    H, Hk, dk, dv, tdt, n = case["H"], case["Hk"], case["dk"], case["dv"], _TORCH[case["dtype"]], case["seqs"]
    M = np.array(_rows(case))
    n_rows = int(M.sum())
    s.M, s.base = M, np.cumsum(M) - M
    s.Q = _normal(gen, (n_rows, Hk * dk), tdt)
    s.K = _normal(gen, (n_rows, Hk * dk), tdt, dk ** -0.5)
    s.V = _normal(gen, (n_rows, H * dv), tdt)
    s.O = torch.zeros_like(s.V)
    # Half lives from one row to a few hundred over the heads; gated ones scatter around them.
    s.decay = -torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda") / H)
    if case["gated"]:
        s.decay = s.decay * torch.exp(_normal(gen, (n_rows, H), torch.float32))
    s.scale = dk ** -0.5
    s.states = _normal(gen, (2 * n, H, dk, dv), torch.float32)
    slots = torch.randperm(2 * n, generator=gen, device="cuda").cpu().numpy()
    s.src = np.full(n, -1) if case["to"] == "fresh" else slots[:n]
    s.dst = slots[n:] if case["to"] == "fork" else slots[:n]
    # Where the rows of every sequence lie, padded to the longest.
    last = np.arange(M.max())
    s.row_of, s.live = _dev(s.base[:, None] + np.minimum(last, M[:, None] - 1)), _dev(last < M[:, None])
    s.from_, s.to = _dev(np.maximum(s.src, 0)), _dev(s.dst)
    s.real = _dev((last < M[:, None]).reshape(-1).nonzero()[0])
    if own:
        from espetero_amd import abi, device
        device.init(0)
        p = device.linear_params(H, Hk, dk, dv, abi.ESP_F16 if case["dtype"] == F16 else abi.ESP_BF16, s.scale, 2 * n, row_decay=case["gated"])
        seqs = np.zeros(n, abi.LINEAR_SEQ_DT)
        seqs["base"], seqs["rows"], seqs["src"], seqs["dst"] = s.base, M, s.src, s.dst
        s.lp = device.LinearPass(p, seqs, n_rows)


def _prepare_shaped(s, case, gen):
    H, Hkv, hd, bt, tdt = case["H"], case["Hkv"], case["hd"], case["bt"], _TORCH[case["dtype"]]
    seqs = _sequences(case)
    n_rows = sum(M for _, M in seqs)
    per = [-(-(P + M) // bt) for P, M in seqs]
    n_blocks = sum(per)
    # The pool in the library's layout: per block and KV head, K [bt][hd], then V in groups of 16 tokens, [bt / 16][hd][16].
    s.pool = _normal(gen, n_blocks * 2 * bt * Hkv * hd, tdt)
    s.blocks = torch.randperm(n_blocks, generator=gen, device="cuda").to(torch.int32)
    s.Q = _normal(gen, (n_rows, H * hd), tdt, 2.0)                    # scores of a few units: some keys count for much more than others
    s.O = torch.zeros_like(s.Q)
    s.slopes = torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda") / H) if case["bias"] else None
    s.scale, s.cap = hd ** -0.5, case["cap"]
    s.P, s.M = np.array([P for P, _ in seqs]), np.array([M for _, M in seqs])
    s.base, s.table = np.cumsum(s.M) - s.M, np.cumsum(per) - np.array(per)
    spans = np.concatenate(_spans(case)).astype(np.int32) if case["docs"] or case["prefix"] else None
    # Where the rows and pages of every sequence lie, padded to the longest, and what the rows see.
    last, pages = np.arange(s.M.max()), np.arange(max(per))
    row_of = s.base[:, None] + np.minimum(last, s.M[:, None] - 1)
    s.row_of = _dev(row_of)
    s.page_of = _dev(s.table[:, None] + np.minimum(pages, np.array(per)[:, None] - 1))
    s.qpos = _dev(s.P[:, None] + np.minimum(last, s.M[:, None] - 1))
    s.real = _dev((last < s.M[:, None]).reshape(-1).nonzero()[0])
    seen = _visible(case)
    s.first, s.end = (_dev(np.concatenate([v[i] for v in seen])[row_of]) for i in (0, 1))
    if own:
        from espetero_amd import abi, device, host, synth
        device.init(0)
        rows = int(s.M.max())
        p = synth.make_params(H, Hkv, hd, abi.ESP_F16 if case["dtype"] == F16 else abi.ESP_BF16, bt, window=case["window"], scale=s.scale,
                              rows_per_tile=rows)
        p.rows_per_tile = device.attn_shaped_rows(p, rows)
        trees, pos = np.zeros(len(seqs), abi.TREE_DT), np.zeros((n_rows, 4), np.int32)
        for i, (P, M) in enumerate(seqs):
            trees[i] = (s.base[i], P, s.table[i], M)
            pos[s.base[i]:s.base[i] + M, :3] = (P + np.arange(M))[:, None]
        resident, groups = device.attn_shaped_hint(p)
        tiles, jobs, n_parts = host.plan_tiles(trees, groups, case["window"], pos if case["window"] else None,
                                               host.options_mi355x(p.rows_per_tile, resident))
        s.sp = device.ShapedPass(p, device.shape_params(s.cap, s.slopes), trees, tiles, jobs, n_parts, n_rows, s.blocks.cpu().numpy(), spans=spans,
                                 pool_blocks=n_blocks)


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(s):
    if s.case["op"] == "linear":
        if own:
            s.lp.run(s.Q, s.K, s.V, s.decay, s.states, s.O)
        else:
            s.O = _plain_linear(s)
        return {"O": s.O, "states": s.states}
    if own:
        s.sp.run(s.Q, s.pool, s.O)
        return s.O
    return _plain_shaped(s)


def _plain_linear(s):
    c = s.case
    H, Hk, dk, dv = c["H"], c["Hk"], c["dk"], c["dv"]
    n, rows = s.row_of.shape
    per = lambda x, heads, d: x[s.row_of].view(n, rows, heads, d).transpose(1, 2).float()  # noqa: E731
    q, k = (per(x, Hk, dk).repeat_interleave(H // Hk, 1) for x in (s.Q, s.K))
    v = per(s.V, H, dv) * s.live[:, None, :, None]
    k = k * s.live[:, None, :, None]
    d = (s.decay[s.row_of] if c["gated"] else s.decay.expand(n, rows, H)).double() * s.live[:, :, None]
    S = s.states[s.from_] if c["to"] != "fresh" else torch.zeros(n, H, dk, dv, device="cuda")
    out = []
    for at in range(0, rows, _CHUNK):
        q_, k_, v_ = (x[:, :, at:at + _CHUNK] for x in (q, k, v))
        sum_ = d[:, at:at + _CHUNK].cumsum(1).transpose(1, 2)                                          # [n][H][rows of the chunk]
        ago = sum_[..., :, None] - sum_[..., None, :]
        below = torch.ones(ago.shape[-2:], dtype=torch.bool, device="cuda").tril()
        weight = torch.exp(torch.where(below, ago, float("-inf"))).float()
        P = torch.matmul(q_, k_.transpose(-1, -2).contiguous()) * weight
        out.append(torch.matmul(P, v_) + torch.exp(sum_).float()[..., None] * torch.matmul(q_, S))
        left = torch.exp(sum_[..., -1:] - sum_).float()
        S = torch.exp(sum_[..., -1:]).float()[..., None] * S + torch.matmul((k_ * left[..., None]).transpose(-1, -2).contiguous(), v_)
    s.states[s.to] = S
    O = torch.cat(out, 2) * s.scale
    return O.transpose(1, 2).reshape(n * rows, H * dv)[s.real].to(s.V.dtype)


def _plain_shaped(s):
    c, d = s.case, s.case["hd"]
    H, Hkv, bt = c["H"], c["Hkv"], c["bt"]
    S, R = s.row_of.shape
    G = H // Hkv
    page = s.pool.view(-1, Hkv, 2, bt * d)[s.blocks.long()[s.page_of]]                              # [S][pages][Hkv][2][bt d]
    L = page.shape[1] * bt
    K = page[:, :, :, 0].reshape(S, -1, Hkv, bt, d).permute(0, 2, 1, 3, 4).reshape(S, Hkv, L, d).float()
    V = page[:, :, :, 1].reshape(S, -1, Hkv, bt // 16, d, 16).permute(0, 2, 1, 3, 5, 4).reshape(S, Hkv, L, d).float()
    Q = s.Q[s.row_of].view(S, R, Hkv, G, d).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * R, d).float()
    x = torch.matmul(Q, K.transpose(-1, -2).contiguous()).view(S, Hkv, G, R, L)
    x *= s.scale
    if s.cap:
        x /= s.cap
        x.tanh_()
        x *= s.cap
    j = torch.arange(L, device="cuda")
    if s.slopes is not None:
        x -= s.slopes.view(Hkv, G, 1, 1) * (s.qpos[:, :, None] - j).abs()[:, None, None].float()
    x.masked_fill_(((j < s.first[:, :, None]) | (j >= s.end[:, :, None]))[:, None, None], float("-inf"))
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    O = torch.matmul(x.view(S, Hkv, G * R, L), V).view(S, Hkv, G, R, d) / total
    return O.permute(0, 3, 1, 2, 4).reshape(S * R, H * d)[s.real].to(s.Q.dtype)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_linear(s) if case["op"] == "linear" else _exact_shaped(s)


def _exact_linear(s):
    """Row by row, as the recurrence says; all sequences at once."""
    c = s.case
    H, Hk, dk, dv = c["H"], c["Hk"], c["dk"], c["dv"]
    O = torch.zeros(s.V.shape, dtype=torch.float64, device="cuda")
    states = s.states.double()
    S = torch.zeros(c["seqs"], H, dk, dv, dtype=torch.float64, device="cuda")
    if c["to"] != "fresh":
        S = states[s.from_].clone()
    order = sorted(range(c["seqs"]), key=lambda i: -s.M[i])                    # those that have a row t come first
    S = S[order]
    base, group = _dev(s.base[order]), H // Hk
    for t in range(int(s.M.max())):
        n = int((s.M > t).sum())
        r = base[:n] + t
        lam = torch.exp((s.decay[r] if c["gated"] else s.decay.expand(n, H)).double())
        q, k = (x[r].view(n, Hk, 1, dk).expand(n, Hk, group, dk).reshape(n, H, dk).double() for x in (s.Q, s.K))
        v = s.V[r].view(n, H, 1, dv).double()
        S[:n] = lam[:, :, None, None] * S[:n] + k[..., None] * v
        O[r] = (q[..., None] * S[:n]).sum(2).view(n, H * dv) * s.scale
    states[s.to[torch.tensor(order, device="cuda")]] = S
    return {"O": O, "states": states}


def _exact_shaped(s):
    c, d = s.case, s.case["hd"]
    H, Hkv, bt = c["H"], c["Hkv"], c["bt"]
    out = torch.zeros(s.Q.shape, dtype=torch.float64, device="cuda")
    pool = s.pool.view(-1, Hkv, 2, bt * d)
    spans = _spans(c)
    for i, (base, P, table, M) in enumerate(zip(s.base.tolist(), s.P.tolist(), s.table.tolist(), s.M.tolist())):
        n = P + M
        pages = pool[s.blocks[table:table + -(-n // bt)].long()]
        p, j = P + torch.arange(M, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        first, prefix = _dev(spans[i][:, :1]), _dev(spans[i][:, 1:])
        seen = (j >= first) & ((j <= p) | (j < prefix))
        if c["window"]:
            seen &= p - j < c["window"]
        for kv in range(Hkv):
            v = pages[:, kv, 1].reshape(-1, d, 16).transpose(1, 2).reshape(-1, d)[:n].double()
            k = pages[:, kv, 0].reshape(-1, d)[:n].double()
            for h in range(kv * (H // Hkv), (kv + 1) * (H // Hkv)):
                x = s.Q[base:base + M, h * d:(h + 1) * d].double() @ k.t() * s.scale
                if s.cap:
                    x = s.cap * torch.tanh(x / s.cap)
                if s.slopes is not None:
                    x = x - float(s.slopes[h]) * (p - j).abs()
                out[base:base + M, h * d:(h + 1) * d] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v
    return out
