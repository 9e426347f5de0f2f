"""Cross attention and its gradients on the GPU, against the definitions in float64 (tests/cross_util.py derives how far
a right kernel may be off)."""
import numpy as np
import pytest

import cross_util as cu
import transfer_station_amd as ts

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module", autouse=True)
def _gpu_present():
    assert ts.device_count() >= 1, "no HIP device visible: GPU tests must run on the MI355X box"


# (sequences of (rows, states), Hq, Hkv, D, room of a padded batch, the states that the call claims to have)
CASES = [
    ([(1, 1)], 1, 1, 16, None, 0),
    ([(1, 300)], 16, 16, 64, None, 0),
    ([(5, 77), (5, 201), (5, 1)], 4, 4, 64, None, 0),
    ([(3, 130), (1, 40)], 32, 8, 128, None, 0),
    ([(33, 50), (20, 129), (1, 7)], 4, 2, 64, None, 0),
    ([(100, 65), (64, 64), (128, 128)], 8, 2, 128, None, 0),
    ([(130, 33), (7, 257)], 2, 1, 256, None, 0),
    ([(40, 100), (90, 31)], 6, 3, 96, (96, 104), 0),
    ([(17, 19), (65, 200)], 4, 4, 80, (70, 210), 0),
    ([(50, 60), (30, 0), (0, 40), (20, 10)], 4, 2, 32, None, 0),
    ([(12, 500), (0, 0), (3, 0)], 8, 1, 192, (12, 500), 0),
    ([(300, 77)], 10, 10, 64, None, 0),
    ([(9, 3000)], 2, 2, 128, None, 0),
    ([(600, 40)], 4, 1, 48, None, 0),
    ([(2, 2000)], 24, 1, 256, None, 0),
    ([(200, 500), (350, 130)], 8, 8, 256, None, 0),
    # many short sequences, some without rows or states: the decode line past its first 64
    ([(b % 3, (37 * b) % 400) for b in range(150)], 4, 2, 64, None, 0),
    ([(1, 300)] * 12, 8, 8, 16, None, 0),
    # two blocks of 16 rows, or two tiles of one, per kv head
    ([(20, 100), (17, 300)], 4, 4, 64, None, 0),
    ([(6, 50), (5, 700), (1, 1)], 16, 4, 128, None, 0),
    ([(16, 300)], 1, 1, 256, None, 0),
    ([(7, 150), (2, 400)], 12, 4, 240, None, 0),
    # the longest of up to 64 sequences first: by their states, equal ones too, and by their rows; one more than 64
    ([(33 + b % 7 * 9, 13 * b * b % 600 // 3 * 3 + (b == 5) * 500) for b in range(64)], 10, 10, 64, None, 0),
    ([(30 * b, 280 - 11 * b) for b in range(21)], 16, 16, 32, None, 0),
    ([(33 + b % 40, 600 - b) for b in range(65)], 8, 8, 64, None, 0),
    # more scores than are taken in two parts
    ([(300, 1100)], 8, 8, 80, None, 0),
    # two teams of waves for dK and dV
    ([(4200, 130)], 16, 16, 64, None, 0),
    ([(2100, 100), (100, 33)], 16, 16, 80, None, 0),
    ([(1500, 70), (300, 200), (0, 20)], 24, 4, 128, None, 0),
    # calls that claim much to read: four kv heads in a workgroup
    ([(1, 900), (1, 130), (1, 2000)], 8, 8, 64, None, 1 << 18),
    ([(5, 300), (4, 700)], 16, 4, 48, None, 1 << 20),
    ([(1, 513), (1, 64), (0, 5)], 32, 8, 128, None, 1 << 18),
    ([(6, 400)], 16, 4, 112, None, 1 << 20),
    ([(1, 700), (1, 3)], 8, 4, 256, None, 1 << 18),
    ([(3, 300)], 32, 4, 176, None, 1 << 18),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_values_and_gradients(case):
    seqs, Hq, Hkv, D, room, claim = CASES[case]
    say("cross", case, CASES[case][1:], seqs[:6])
    t = cu.Batch(seqs, Hq, Hkv, D, 100 * case + 1, room, claim)
    cu.check(t, cu.run(t), cu.reference(t), "case %d" % case)
