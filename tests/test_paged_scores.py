"""Scores of the paged attention over the whole range of what a caller may ask for: score caps from a fraction of the
scores to far above them, with bounds that do not grow with the cap."""
import numpy as np
import pytest

import paged_util as pu
from test_paged import check


# One of each kernel: bits, D, page, Hq, Hkv, (new, length) by sequence. One and two row blocks of the decode kernel
# at each slot of head dims, 64 rows on key halves, eight waves on key halves, tiles of 128 rows.
CALLS = [
    (16, 64, 16, 8, 2, [(1, 700), (1, 33)]),
    (16, 128, 64, 8, 1, [(2, 600), (1, 90)]),
    (16, 256, 32, 8, 2, [(1, 300), (3, 40)]),
    (4, 64, 16, 4, 2, [(1, 500)]),
    (4, 128, 32, 8, 2, [(1, 400), (4, 60)]),
    (4, 256, 64, 8, 2, [(1, 410)]),
    (16, 128, 32, 8, 2, [(7, 300)]),
    (4, 64, 32, 4, 1, [(5, 260)]),
    (16, 128, 16, 8, 1, [(8, 500)]),
    (4, 128, 64, 16, 2, [(7, 300)]),
    (16, 64, 32, 6, 3, [(70, 333)]),
    (4, 128, 16, 4, 1, [(50, 260)]),
    (16, 256, 32, 4, 2, [(70, 140)]),
    (4, 256, 32, 4, 1, [(80, 130)]),
]
CAPS = [0.5, 40.0, 256.0, 257.0, 2e3, 1e4, 1e5, 1e6]


def scores_ref(c, q, Hq, scale, cap, terms=None):
    """(O, bound) in float64. The bound follows the roundings as attend_ref's does, with P's and O's 2^-8, exp2's 2^-21
    and a rounding of 2^-24 per key in the sums, but takes the cap's error from the score itself. With s the score
    and t = cap tanh(s / cap), dt/ds <= 1, so the D + 8 roundings of the product (terms + 8 where only so many of a
    row's elements are not zero) count as they are, 2^-24 of scale |q|.|k| each. tanh itself is allowed 32 roundings of t, and up to a cap of 256 a formula whose error goes by
    the cap: cap (1 - 2 r), r = 1 / (2^x + 1) <= 1 from an exp2 and a reciprocal good to 2^-23 each and three
    roundings of 2^-24, so 7 2^-24 of 2 r cap, under 2^-20 cap; at 256 that is 2^-12, a sixteenth of P's 2^-8."""
    D, g = c.D, Hq // c.Hkv
    O, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b, (n, kv) in enumerate(c.seqs):
        K, V = c.get(b, 0, kv)
        r = slice(c.start[b], c.start[b] + n)
        show = np.arange(kv)[None, :] <= kv - n + np.arange(n)[:, None]
        for h in range(Hq):
            x, k, v = pu.f32(q[r, h]).astype(np.float64), K[:, h // g], V[:, h // g]
            s = scale * (x @ k.T)
            t = cap * np.tanh(s / cap)
            off = ((terms or D) + 8) * 2.0 ** -24 * scale * (np.abs(x) @ np.abs(k).T) + 32 * 2.0 ** -24 * np.abs(t)
            off = np.where(show, off + (2.0 ** -20 * cap if cap <= 256 else 0.0), 0.0).max(1)
            t = np.where(show, t, -np.inf)
            w = np.exp(t - t.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            delta = 2 * (off + 2.0 ** -21 * (kv / 32 + 2))
            O[r, h] = w @ v
            bound[r, h] = 2.0 ** -8 * np.abs(O[r, h]) + (w @ np.abs(v)) * (
                2.0 ** -8 * 1.01 + delta[:, None] + kv * 2.0 ** -24) + 1e-30
    return O, bound


@pytest.mark.gpu
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("case", CALLS, ids=["%d-%d-%d" % (c[0], c[1], i) for i, c in enumerate(CALLS)])
def test_caps_of_any_size(case, cap):
    """A cap far above the scores leaves them as they are; at and below them it bends them."""
    bits, D, page, Hq, Hkv, seqs = case
    print("cap", case, cap, flush=True)
    c = pu.Cache(seqs, Hkv, D, page, bits, 3)
    c.fill(31)
    q = pu.normal((c.N, Hq, D), 5, 2.0)
    ref, bound = scores_ref(c, q, Hq, D ** -0.5, cap)
    check(pu.attend(c, q, Hq, 1, 0.0, cap), ref, bound, (case, cap))


@pytest.mark.gpu
@pytest.mark.parametrize("cap,sigma", [(257.0, 160.0), (1e4, 4000.0)])
@pytest.mark.parametrize("bits,n", [(16, 1), (4, 1), (16, 8), (16, 90), (4, 90)])
def test_scores_on_both_sides_of_a_large_cap(bits, n, cap, sigma):
    """Rows whose largest scores lie from a hundredth of the cap to its double, on both sides of the quarter where one
    form of tanh ends, with scores one apart beside them: an error of a thousandth of the cap shows."""
    D, page, kv = 128, 32, 400
    c = pu.Cache([(n, kv)], 1, D, page, bits, 3)
    K, V = np.zeros((kv, 1, D), np.float32), pu.normal((kv, 1, D), 2)
    j = np.arange(kv)
    # Two columns hold the score: a coarse part and a fine one, exact in bf16 and in 4 bits.
    K[:, 0, 0] = np.array([0.5, 1, 1.5, 2, 3, 4, 6])[j % 7]
    K[:, 0, 32] = np.array([0.5, 1, 1.5, 2, 3, 4, 6])[j // 7 % 7]
    c.put(0, 0, pu.bf16(K), V)
    q = np.zeros((n, 2, D), np.float32)
    rows = np.random.default_rng(1).uniform(0.02, 1.0, (n, 2))
    q[:, :, 0] = sigma * rows * D ** 0.5 / 2
    q[:, :, 32] = 2.0 * D ** 0.5
    q = pu.bf16(q)
    ref, bound = scores_ref(c, q, 2, D ** -0.5, cap, terms=2)
    check(pu.attend(c, q, 2, 1, 0.0, cap), ref, bound, (bits, n, cap))


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [30.0, 1e4])
@pytest.mark.parametrize("bits,n,kv", [(16, 1, 100), (4, 1, 3000), (16, 8, 900), (4, 20, 700), (16, 100, 600), (4, 40, 96)])
def test_nan_and_infinities_under_a_cap(bits, n, kv, cap):
    """An infinity in a row of q gives scores of the cap and its negative; a NaN there, or in a key, makes NaN of the
    rows that meet it and of no other."""
    Hq, Hkv, D = 4, 2, 128
    c = pu.Cache([(n, kv), (n, kv // 2)], Hkv, D, 32, bits, 3)
    c.fill(23)
    for b, m in ((0, kv), (1, kv // 2)):  # the column that meets the infinity: half the keys on either side
        K, V = ([pu.bf16(x.astype(np.float32)) for x in c.get(b, 0, m)])
        K[:, :, 64:96] = pu.bf16(np.where(np.arange(m) % 2, 1.0, -1.0)[:, None, None] * np.ones((m, Hkv, 32), np.float32))
        c.put(b, 0, K, V)
    pg, at = c.places(0, kv - (n + 1) // 2, kv)
    x, nan = (c.ks, 255) if bits == 4 else (c.k, 0xFF)
    x[pg[0], 1, at[0]] = nan
    q = pu.normal((c.N, Hq, D), 5)
    q[c.N - 1, 0, 70], q[c.N - 1, 1, 70] = 0x7F80, 0xFF80  # inf and -inf, which meet kv head 0
    q[0, 0, 5] = 0x7FC0  # NaN
    with np.errstate(invalid="ignore"):
        ref, bound = scores_ref(c, q, Hq, D ** -0.5, cap)
    lost = np.isnan(ref).any(-1)
    assert lost[0, 0] and lost.sum() == 1 + 2 * ((n + 1) // 2) and not lost[c.N - 1].any()
    # the infinities' rows: every other key they see, alike, whatever the product's roundings
    m = kv // 2
    V = c.get(1, 0, m)[1][:, 0]
    for h, keys in ((0, V[1::2]), (1, V[0::2])):
        bound[c.N - 1, h] = (2.0 ** -8 * np.abs(keys.mean(0)) + np.abs(keys).mean(0) * (2.0 ** -8 * 1.01 + m * 2.0 ** -24 +
                                                                                   2 * 2.0 ** -20 * min(cap, 256)))
        ref[c.N - 1, h] = keys.mean(0)
    O = pu.attend(c, q, Hq, 1, 0.0, cap, poison=0x3F)
    assert np.array_equal(np.isnan(O).any(-1), lost) and np.array_equal(np.isnan(O).all(-1), lost)
    check(np.where(lost[..., None], 0, O), np.where(lost[..., None], 0, ref), np.where(lost[..., None], 0, bound),
          (bits, n, kv, cap))


@pytest.mark.gpu
@pytest.mark.parametrize("bits,n", [(16, 1), (4, 1), (16, 8), (16, 40), (4, 90)])
@pytest.mark.parametrize("top", [16, 24, 29])
def test_scores_up_to_two_to_the_thirtieth(bits, n, top):
    """One key of a score of 2^top and others of three quarters of it and less: each row is that key's V to the
    rounding of P and O, wherever the key lies and however the roundings of such scores fall."""
    D, page, kv = 64, 32, 1500
    K, V = np.zeros((kv, 1, D), np.float32), pu.normal((kv, 1, D), 2)
    K[:, 0, 0] = np.array([0.5, 1, -1, 2, -3, 4, 1.5])[np.arange(kv) % 7]
    K[0, 0, 1] = 6.0  # the scales of all groups alike in 4 bits
    for at in (0, 31, 128, 700, kv - n - 1):
        k = K.copy()
        k[at, 0, 0] = 6.0
        c = pu.Cache([(n, kv)], 1, D, page, bits, 3)
        c.put(0, 0, pu.bf16(k), V)
        q = np.zeros((n, 2, D), np.uint16)
        q[:, :, 0] = pu.bf16(np.float32(2.0 ** top / 6.0 * D ** 0.5))
        O = pu.attend(c, q, 2, 1)
        v = c.get(0, at, at + 1)[1][0, 0]
        check(O, np.broadcast_to(v, O.shape), np.broadcast_to(2 * 2.0 ** -8 * 1.01 * np.abs(v), O.shape), (bits, n, top, at))


def large_scores(bits, D, Hq, kv, levels, rows_q0, page=256, n=1):
    """(cache, q, reference, bound): scores of about 2^20 that fp32 holds exactly. Column 0 gives every key the same
    large score, a power of two times 1 to 2 by the row's q; column 32 adds twice the key's level (in 0, 0.5 .. 6, which
    4 bits hold). D is 64 or 256, so that 1/sqrt(D) is a power of two and all products and sums are exact; what is left
    are the roundings of P and O and of exp2: 2^-21 once per weight and once per rescale, and 2^-22 of the distance to
    the row's largest score, for log2(e)'s."""
    r = int(D ** 0.5)
    K, V = np.zeros((kv, 1, D), np.float32), pu.normal((kv, 1, D), 2)
    K[:, 0, 0], K[:, 0, 32] = 4.0, levels
    c = pu.Cache([(n, kv)], 1, D, page, bits, 3)
    c.put(0, 0, pu.bf16(K), V)
    q = np.zeros((n, Hq, D), np.float32)
    q[:, :, 0], q[:, :, 32] = 2.0 ** 20 / 4 * r * rows_q0, 2.0 * r
    q = pu.bf16(q)
    v = c.get(0, 0, kv)[1][:, 0]
    t = 2.0 * levels.astype(np.float64)
    w = np.exp(t - t.max())
    w /= w.sum()
    ref, A = w @ v, w @ np.abs(v)
    delta = 2 * (2.0 ** -22 * (t.max() - t.min()) + 2.0 ** -21 * (4 + 2))
    bound = 2.0 ** -8 * np.abs(ref) + A * (2.0 ** -8 * 1.01 + delta + 2.0 ** -12)
    return c, q, np.broadcast_to(ref, q.shape), np.broadcast_to(bound, q.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,D,Hq,kv", [(16, 64, 8, 1600), (4, 64, 8, 1600), (16, 256, 8, 1600), (4, 256, 8, 1600),
                                          (16, 64, 24, 1600), (16, 64, 64, 160000), (16, 64, 128, 160000),
                                          (4, 64, 128, 160000), (16, 256, 128, 160000)])
def test_keys_before_a_rise_keep_their_weight(bits, D, Hq, kv):
    """A maximum that rises late, at scores of 2^20: the keys before, as many as outweigh the step, count as much as the
    key that raises it, to the rounding of P. No parts (T is large), so that one workgroup sees all keys in turn."""
    levels = np.zeros(kv)
    j = np.arange(kv)
    if kv == 1600:  # decode: a step of e^6 against 416 keys, all of the one wave whose maximum rises
        levels[(j % 128 < 32) & (j < 1536)] = 3.0
        levels[1536:1568] = 0.0
        levels[1541] = 6.0
    else:  # prefill: a step of e^12
        levels[kv - 70] = 6.0
    c, q, ref, bound = large_scores(bits, D, Hq, kv, levels, 1 + np.arange(Hq) % 64 / 64)
    O = pu.attend(c, q, Hq, 0, pad=40000 // Hq)
    check(O, ref, bound, (bits, D, Hq))


@pytest.mark.gpu
@pytest.mark.parametrize("bits,D,Hq", [(16, 64, 8), (4, 64, 8), (4, 256, 8), (16, 64, 24), (16, 64, 64), (4, 64, 64),
                                       (16, 64, 128), (4, 64, 128), (16, 256, 128)])
def test_parts_and_halves_keep_their_weight(bits, D, Hq):
    """Parts, key halves and waves whose maxima differ a little, at scores of 2^20, joined by what they are."""
    kv = 6000
    levels = np.array([0, 0.5, 1, 1.5, 2])[np.random.default_rng(3).integers(0, 5, kv)]
    step = np.repeat(np.random.default_rng(4).integers(0, 3, kv // 16), 16) * 0.5
    levels = np.where(levels + step > 2, 2.0, levels + step)
    levels[np.arange(kv) % 1024 < 300] = 0.0
    c, q, ref, bound = large_scores(bits, D, Hq, kv, levels, 1 + np.arange(Hq) % 64 / 64)
    check(pu.attend(c, q, Hq, 0), ref, bound, (bits, D, Hq))


def test_the_bound_tells_a_cap_apart_that_loses_small_scores():
    """The bound of these tests against cap (1 - 2 / (2^x + 1)) taken in float32 throughout: it holds for a cap of 40,
    and not for 1e6."""
    D, kv, Hq = 128, 600, 8
    c = pu.Cache([(2, kv)], 1, D, 64, 16, 3)
    c.fill(31)
    q = pu.normal((2, Hq, D), 5, 2.0)
    for cap, held in ((40.0, True), (1e6, False)):
        ref, bound = scores_ref(c, q, Hq, D ** -0.5, cap)
        K, V = c.get(0, 0, kv)
        s = np.einsum("nhd,jd->nhj", pu.f32(q).astype(np.float64), K[:, 0]).astype(np.float32)
        cap_in = np.float32(2 * np.log2(np.e) * D ** -0.5 / cap)
        cap_out = np.float32(cap * np.log2(np.e))
        t = cap_out - np.float32(2) * cap_out / (np.exp2(s * cap_in) + np.float32(1))
        t = np.where(np.arange(kv) <= kv - 2 + np.arange(2)[:, None, None], t.astype(np.float64), -np.inf)
        w = np.exp2(t - t.max(-1, keepdims=True))
        O = np.einsum("nhj,jd->nhd", w / w.sum(-1, keepdims=True), V[:, 0])
        assert bool(np.all(np.abs(O - ref) <= bound)) == held, cap
