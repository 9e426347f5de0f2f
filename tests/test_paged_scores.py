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
