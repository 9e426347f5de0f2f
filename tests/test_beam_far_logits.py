"""Selection over logits so large, or so low, that the logarithm of their sum is lost beside them: log-softmax does not
change when all logits of a row are moved alike."""
import numpy as np
import pytest

import test_beam
import transfer_station_amd as ts
from paged_util import bf16, f32

LOWEST = {16: float(f32(np.array([0xFF7F], np.uint16))[0]), 32: float(np.finfo(np.float32).min)}


def select_ref(x, scores, B, beams, K):
    """As test_beam.select_ref, by (x - top) - log sum exp(x - top)."""
    V, n = x.shape[1], min(K, x.shape[1])
    out = np.full((B, K), -np.inf), np.full((B, K), -1), np.repeat(beams * np.arange(B)[:, None], K, 1)
    for b in range(B):
        c, tok = np.zeros((beams, n)), np.zeros((beams, n), int)
        for i in range(beams):
            r = b * beams + i
            d = x[r] - x[r].max()
            tok[i] = np.argsort(-x[r], kind="stable")[:K]
            c[i] = (d[tok[i]] - np.log(np.exp(d).sum())) + float(scores[r])
        best = np.argsort(-c.reshape(-1), kind="stable")[:K]
        out[0][b, :len(best)], out[1][b, :len(best)] = c.reshape(-1)[best], tok.reshape(-1)[best]
        out[2][b, :len(best)] = b * beams + best // n
    return out


def run(x, scores, bits, B, beams, K):
    logits = bf16(x) if bits == 16 else x
    return test_beam.select(logits, scores, None, 0, B, beams, x.shape[1], K)


def test_reference_does_not_change_with_the_place_of_the_logits():
    """In fp64 the test's own definition gives 1/V to each of V equal logits of any size, and moved rows the same."""
    for value in (0.0, 1e30, LOWEST[32], LOWEST[16]):
        got = select_ref(np.full((1, 50), value), np.zeros(1), 1, 1, 7)
        assert np.allclose(got[0], -np.log(50), rtol=1e-14) and np.array_equal(got[1][0], np.arange(7))
    x = np.random.default_rng(1).integers(-9, 9, (2, 40)).astype(np.float64)
    for a, b in zip(select_ref(x, np.zeros(2), 1, 2, 9), select_ref(x + 2.0 ** 40, np.zeros(2), 1, 2, 9)):
        assert np.array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("V", [7, 600, 40000])
@pytest.mark.parametrize("value", [0.0, 1e30, -1e30, 2.0 ** 60, "lowest"])
def test_equal_logits_of_any_size(value, V, bits):
    assert ts.device_count() >= 1
    print("equal", value, V, bits, flush=True)
    v = LOWEST[bits] if value == "lowest" else float(f32(bf16(np.array([value], np.float32)))[0])
    x = np.full((2, V), v, np.float32)
    scores = np.array([-1.5, -1.25], np.float32)
    got = run(x, scores, bits, 1, 2, 6)
    assert np.allclose(got[0], -1.25 - np.log(V), rtol=2.0 ** -20, atol=0)
    test_beam.check_select(got, select_ref(x.astype(np.float64), scores, 1, 2, 6))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("V", [600, 40000])
def test_a_masked_beam_does_not_win(V, bits):
    """Beams without, with few and with all logits left, the rest at the type's lowest value; K of more than are left."""
    assert ts.device_count() >= 1
    print("masked", V, bits, flush=True)
    B, beams, K, low = 3, 4, 16, LOWEST[bits]
    x = f32(bf16(np.random.default_rng(V).standard_normal((B * beams, V)).astype(np.float32) * 2)).copy()
    x[1] = low                       # beside beams with all their logits
    x[4:8] = low
    x[4, 11], x[6, [5, V - 2]] = 3.0, (1.0, 0.5)  # two beams of few, two of none
    x[8:12, 3:] = low                # twelve left for sixteen: masked tokens follow at their own score
    scores = (-np.arange(B * beams)).astype(np.float32)
    scores[9] = -100.0
    got = run(x, scores, bits, B, beams, K)
    ref = select_ref(x.astype(np.float64), scores, B, beams, K)
    test_beam.check_select(got, ref)
    assert 1 not in got[2][0] or got[0][0][got[2][0] == 1].max() <= -1 - np.log(V) + 1e-5
    assert np.all(np.diff(got[0], axis=1) <= 0)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 32])
def test_rows_moved_by_a_large_number(bits):
    """Multiples of 2^35 moved by 2^41 (exact in both types' rows here): the scores of rows that are not moved."""
    assert ts.device_count() >= 1
    rng = np.random.default_rng(8)
    V, K = 3000, 20
    unit = np.float32(2.0 ** 35)
    x = (rng.integers(-30, 30, (4, V)) * unit).astype(np.float32)
    x[1] += np.float32(2.0 ** 41)
    x[3] -= np.float32(2.0 ** 41)
    assert np.array_equal(f32(bf16(x)), x)
    scores = np.array([0, -0.5, 0.25, -0.125], np.float32)
    test_beam.check_select(run(x, scores, bits, 2, 2, K), select_ref(x.astype(np.float64), scores, 2, 2, K))
