"""esp_attn_shaped on the device: the weights' second 16 bits reach the product with V, and infinite values are no less infinite for it."""
import numpy as np
import pytest

from shaped_precision import bound
from shaped_utils import ShapedCase, documents
from test_gpu_shaped import Run, dev
from espetero_amd import abi, synth
from oracle import binding as ob

pytestmark = pytest.mark.gpu

F16, BF16 = abi.ESP_F16, abi.ESP_BF16


def check(c, rows=None, shift=0, **plan):
    r = Run(c, **plan)
    want, tol, which = bound(c, shift, rows)
    got = ob.to_f32(r()[which][:, :c.H * c.hd], c.dtype).astype(np.float64).reshape(want.shape)
    print(f"  of the bound: {np.max(np.abs(got - want) / tol):.3f}", flush=True)
    assert np.all(np.abs(got - want) <= tol)


SHAPES = [(0.0, False), (20.0, False), (0.0, True), (30.0, True)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cap,bias", SHAPES)
@pytest.mark.parametrize("heads,hd,seqs", [((8, 2), 128, [(40, 1), (130, 1)]), ((4, 2), 128, [(200, 16)]), ((8, 2), 256, [(60, 2), (200, 4)])])
def test_few_rows_hold_their_weights_as_two_numbers(heads, hd, seqs, cap, bias, dtype):
    c = ShapedCase(*heads, hd, dtype, 16, seqs, cap=cap, bias=bias, sharp=0.25, seed=hd)
    check(c)
    check(c, workgroups=4096)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cap,bias", SHAPES)
@pytest.mark.parametrize("heads,hd,seqs", [((8, 2), 128, [(0, 150), (333, 70)]), ((4, 4), 128, [(500, 40)]), ((4, 2), 256, [(0, 150), (333, 70)])])
def test_many_rows_hold_their_weights_as_two_numbers(heads, hd, seqs, cap, bias, dtype):
    c = ShapedCase(*heads, hd, dtype, 16, seqs, cap=cap, bias=bias, sharp=0.25, seed=hd)
    check(c, range(0, 150, 7))
    check(c, range(0, 150, 7), workgroups=2048, cut_batch=True)


@pytest.mark.parametrize("hd", [128, 256])
def test_many_rows_of_documents_hold_their_weights_as_two_numbers(hd):
    """Stages that some rows see in part."""
    c = ShapedCase(4, 2, hd, BF16, 16, [(45, 150)], spans=[documents(45, 150, [0, 90, 100, 160], 40)], cap=20.0, bias=True, sharp=0.25, seed=hd)
    check(c, range(0, 150, 5))


def with_values(c, values):
    """The pool with `values` ({(key, KV head, dim): bits}) in the first sequence's V."""
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * c.hd)
    for (j, kvh, dim), bits in values.items():
        b, t = c.block_list[j // c.bt], j % c.bt
        pool[b, kvh, 1].reshape(c.bt // 16, c.hd, 16)[t // 16, dim, t % 16] = bits
    return dev(pool.reshape(-1))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,cap,bias", [(128, 0.0, False), (128, 20.0, True), (256, 0.0, True), (256, 20.0, False)])
@pytest.mark.parametrize("cut", [False, True])
def test_infinite_values_that_many_rows_see(cut, hd, cap, bias, dtype):
    """Far in front of the rows, where stages are seen whole, also where a weight is nothing beside the largest: an infinity of either sign, both (NaN),
    and one among the rows, which some of them see. Other dims are as exact as ever, other KV heads keep their bits."""
    P, M = 900, 70
    c = ShapedCase(4, 2, hd, dtype, 16, [(P, M)], cap=cap, bias=bias, sharp=0.25, seed=3)
    if bias:
        c.slopes[:2] = 0.5, 2.0                                        # 2^-900 and less at key 100
    inf = 0x7C00 if dtype == F16 else 0x7F80
    r = Run(c, **(dict(workgroups=2048, cut_batch=True) if cut else {}))
    clean = r().reshape(M, 4, hd)
    r.pool = with_values(c, {(100, 0, 3): inf, (411, 0, 40): inf | 0x8000, (100, 0, 77): inf, (700, 0, 77): inf | 0x8000, (P + 50, 0, 90): inf})
    r.O.fill_(0x1234)
    bits = r().reshape(M, 4, hd)
    got = ob.to_f32(bits, dtype)
    assert (got[:, :2, 3] == np.inf).all() and (got[:, :2, 40] == -np.inf).all() and np.isnan(got[:, :2, 77]).all()
    assert (got[50:, :2, 90] == np.inf).all() and np.isfinite(got[:50, :2, 90]).all()
    assert (bits[:, 2:] == clean[:, 2:]).all()
    want, tol, _ = bound(c)
    tol, want = tol[:, :2], want[:, :2]
    odd = ~np.isfinite(got[:, :2])
    assert odd.sum() == 2 * (3 * M + 20)
    assert np.all(odd | (np.abs(got[:, :2] - want) <= tol))


def test_rows_that_meet_no_infinite_value_keep_their_bits():
    """A NaN key of the first document: the rows of the second, of the same tile, are not walked again."""
    P, M = 700, 32
    first = 200
    spans = [[(0 if m < 5 else first, 0) for m in range(M)]]
    c = ShapedCase(4, 1, 128, BF16, 16, [(P, M)], spans=spans, cap=30.0, seed=4)
    r = Run(c)
    clean = r()
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt * c.hd)
    pool[c.block_list[3], 0, 0, 5] = 0x7FC0
    r.pool = dev(pool.reshape(-1))
    r.O.fill_(0x1234)
    bits = r()
    assert (bits[5:] == clean[5:]).all() and np.isnan(ob.to_f32(bits[:5], BF16)).all()


def test_a_value_whose_weight_has_vanished_is_still_infinite():
    """fp16, a key whose weight is 2^-47 of the largest of its part and 2^-200 of the row's, in a stage that one row does not see whole."""
    c = ShapedCase(4, 4, 128, F16, 16, [(600, 40)], bias=True, spans=[[(0, 0)] * 39 + [(9, 0)]], seed=6)
    c.slopes[:] = 0.25
    for plan in (dict(workgroups=4096, cut_batch=True), {}):
        r = Run(c, **plan)
        clean = r().reshape(40, 4, 128)
        r.pool = with_values(c, {(8, 0, 3): 0x7C00, (8, 0, 60): 0xFC00})
        r.O.fill_(0x1234)
        bits = r().reshape(40, 4, 128)
        got = ob.to_f32(bits, F16)
        assert (got[:-1, 0, 3] == np.inf).all() and (got[:-1, 0, 60] == -np.inf).all()
        assert (bits[-1] == clean[-1]).all() and (bits[:, 1:] == clean[:, 1:]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,hd,M,cap,bias", [((4, 2), 128, 1, 0.0, False), ((4, 2), 128, 4, 20.0, True), ((8, 2), 128, 8, 0.0, True), ((4, 2), 256, 1, 0.0, True),
                                                 ((8, 2), 256, 4, 20.0, False)])
@pytest.mark.parametrize("workgroups", [None, 24])
def test_infinite_values_that_few_rows_see(workgroups, heads, hd, M, cap, bias, dtype):
    """Whole tiles and parts: an infinity of either sign, both (NaN), one whose weight is nothing beside the largest, and one among the rows. Whatever meets
    none of them keeps its bits."""
    P, G = 900, heads[0] // heads[1]
    c = ShapedCase(*heads, hd, dtype, 16, [(P, M)], cap=cap, bias=bias, seed=3)
    if bias:
        c.slopes[:G] = 2.0                                             # 2^-2300 at key 100
    inf = 0x7C00 if dtype == F16 else 0x7F80
    r = Run(c, workgroups=workgroups)
    clean = r().reshape(M, heads[0], hd)
    r.pool = with_values(c, {(100, 0, 3): inf, (411, 0, 40): inf | 0x8000, (100, 0, 77): inf, (700, 0, 77): inf | 0x8000, (P + M // 2, 0, 90): inf,
                             (896, 0, 91): inf | 0x8000})
    r.O.fill_(0x1234)
    bits = r().reshape(M, heads[0], hd)
    got = ob.to_f32(bits, dtype)
    assert (got[:, :G, 3] == np.inf).all() and (got[:, :G, 40] == -np.inf).all() and np.isnan(got[:, :G, 77]).all()
    assert (got[M // 2:, :G, 90] == np.inf).all() and (got[:, :G, 91] == -np.inf).all()
    same = np.ones(bits.shape, bool)
    same[:, :G, [3, 40, 77, 91]] = False
    same[M // 2:, :G, 90] = False
    assert (bits[same] == clean[same]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("n", [3000, 30000])
@pytest.mark.parametrize("M,at", [(1, 7), (1, -9), (3, -9), (40, 7), (40, -50)])
def test_many_small_weights_beside_a_large_one(M, at, n, hd, dtype):
    """A flat tail of keys, each of 2^-24.5 of one key's weight (first or last of those that all rows see), whose large values make half of the
    output: fp16 numbers of the largest weight 1 have no half step there."""
    c = ShapedCase(1, 1, hd, dtype, 16, [(n, M)], seed=n)
    at = at if at > 0 else n + at
    f, to = lambda x: ob.to_f32(x, dtype), lambda x: synth._bits(np.atleast_1d(np.asarray(x, np.float32)), dtype)  # noqa: E731
    c.Q[:, :] = 0
    c.Q[:, 0] = to(16.0)[0]
    c.K[0][:] = 0
    c.K[0][at, 0, 0] = to(24.5 * np.log(2) / (16.0 * c.scale))[0]
    rng = np.random.default_rng(n)
    c.V[0][:] = to(rng.uniform(0.5, 1.0, c.V[0].shape) * 2.0 ** 24.5 / n)
    c.V[0][at] = to(rng.uniform(0.5, 1.0, c.V[0][at].shape))
    pool = c.pool.reshape(c.n_blocks, 2, c.bt * hd)
    for b in range(-(-(n + M) // 16)):
        k, v = (x[0][16 * b:16 * b + 16, 0] for x in (c.K, c.V))
        block = pool[c.block_list[b]]
        block[0].reshape(16, hd)[:len(k)] = k
        block[1].reshape(hd, 16)[:, :len(v)] = v.T
    assert f(c.V[0]).max() < 60000
    check(c, range(0, M, 13), shift=15 if M < 40 else 7)
    check(c, range(0, M, 13), shift=15 if M < 40 else 7, workgroups=16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,hd,M", [((4, 2), 128, 70), ((4, 2), 256, 40), ((4, 2), 128, 3)])
def test_infinite_values_of_every_key(heads, hd, M, dtype):
    """A dim of KV head 0 that is infinite for every key, the other KV head NaN throughout; two documents and a prefix."""
    P, inf = 300, 0x7C00 if dtype == F16 else 0x7F80
    c = ShapedCase(*heads, hd, dtype, 32, [(P, M)], spans=[documents(P, M, [0, 60, P + M // 2], 50)], bias=True, sharp=0.25, seed=11)
    r = Run(c)
    pool = c.pool.copy().reshape(c.n_blocks, c.Hkv, 2, c.bt // 16, hd * 16)
    V = pool[:, :, 1].reshape(c.n_blocks, c.Hkv, c.bt // 16, hd, 16)
    V[:, 0, :, 17], V[:, 1] = inf | 0x8000, 0x7E00 if dtype == F16 else 0x7FC0
    pool[:, :, 1] = V.reshape(c.n_blocks, c.Hkv, c.bt // 16, hd * 16)
    r.pool = dev(pool.reshape(-1))
    got = ob.to_f32(r(), dtype).reshape(M, 4, hd)
    want, tol, _ = bound(c)
    assert np.isnan(got[:, 2:]).all() and (got[:, :2, 17] == -np.inf).all()
    keep = np.arange(hd) != 17
    assert np.all(np.abs(got[:, :2, keep] - want[:, :2, keep]) <= tol[:, :2, keep])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (0.0, True), (1.0, False), (1.0, True)])
@pytest.mark.parametrize("hd,M", [(128, 1), (128, 80), (256, 3), (256, 80)])
@pytest.mark.parametrize("scale", [20, 27, 30, 40, 60, 64])
def test_scores_beyond_what_fp32_tells_apart(scale, hd, M, cap, bias, dtype):
    """Scores of 2^20 to 2^69, with caps a hundredth of that or none: rows stay finite and between the values they see, and a row whose largest score is far
    ahead of the others has that key's value."""
    c = ShapedCase(4, 2, hd, dtype, 16, [(700, M)], cap=0.0, bias=bias, seed=21)
    c.scale = 2.0 ** scale
    c.cap = 0.1 * c.scale * cap
    if bias:
        c.slopes *= np.float32(2.0 ** (scale - 8))
    for plan in ({}, dict(workgroups=2048, cut_batch=True)):
        got = ob.to_f32(Run(c, **plan)(), dtype).astype(np.float64).reshape(M, 4, hd)
        assert np.isfinite(got).all()
        for m in (0, M - 1):
            for h in range(4):
                K, V = (ob.to_f32(x[0], dtype).astype(np.float64)[:700 + m + 1, h // 2] for x in (c.K, c.V))
                assert (np.abs(got[m, h]) <= np.abs(V).max(0) * (1 + 2.0 ** -7)).all()
                x = K @ ob.to_f32(c.Q, dtype).astype(np.float64)[m, h * hd:(h + 1) * hd] * c.scale
                x = c.cap * np.tanh(x / c.cap) if c.cap else x
                x = x - (float(c.slopes[h]) * (700 + m - np.arange(700 + m + 1)) if bias else 0)
                top = np.argsort(x)[-2:]
                if x[top[1]] - x[top[0]] > 2.0 ** -10 * np.abs(x).max() + 200:
                    assert (np.abs(got[m, h] - V[top[1]]) <= 2.0 ** -7 * np.abs(V).max(0)).all()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("P", [40, 600])
def test_rows_beside_others_of_any_scores(P, hd, bias):
    """Rows of a tile whose scores are beyond 2^20, infinite or NaN, or whose largest come late: the others are as exact as ever, and where no stage is
    seen whole by all of them they keep their bits."""
    M = 24
    c = ShapedCase(8, 2, hd, BF16, 16, [(P, M)], bias=bias, seed=31)
    r = Run(c, workgroups=1)
    clean = r()
    odd = [1, 2, 9, 16, 23]
    Q = c.Q.copy()
    for m, by in zip(odd, [2.0 ** 24, 2.0 ** 40, 30.0, 8.0, 1.0]):
        Q[m] = synth._bits(ob.to_f32(Q[m], BF16) * np.float32(by), BF16)
    Q[odd[0], 5], Q[odd[4], 7] = 0x7F80, 0x7FC0                          # an infinity, NaN
    r.Q = dev(Q)
    r.O.fill_(0x1234)
    bits = r()
    keep = np.setdiff1d(np.arange(M), odd)
    if P == 40:
        assert (bits[keep] == clean[keep]).all()
    want, tol, _ = bound(c, 0, keep)
    assert np.all(np.abs(ob.to_f32(bits[keep], BF16).reshape(want.shape) - want) <= tol)
