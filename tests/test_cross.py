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


# (sequences of (rows, states), Hq, Hkv, D, room)
CASES = [
    ([(1, 1)], 1, 1, 16, None),
    ([(1, 300)], 16, 16, 64, None),
    ([(5, 77), (5, 201), (5, 1)], 4, 4, 64, None),
    ([(3, 130), (1, 40)], 32, 8, 128, None),
    ([(33, 50), (20, 129), (1, 7)], 4, 2, 64, None),
    ([(100, 65), (64, 64), (128, 128)], 8, 2, 128, None),
    ([(130, 33), (7, 257)], 2, 1, 256, None),
    ([(40, 100), (90, 31)], 6, 3, 96, (96, 104)),
    ([(17, 19), (65, 200)], 4, 4, 80, (70, 210)),
    ([(50, 60), (30, 0), (0, 40), (20, 10)], 4, 2, 32, None),
    ([(12, 500), (0, 0), (3, 0)], 8, 1, 192, (12, 500)),
    ([(300, 77)], 10, 10, 64, None),
    ([(9, 3000)], 2, 2, 128, None),
    ([(600, 40)], 4, 1, 48, None),
    ([(2, 2000)], 24, 1, 256, None),
    ([(200, 500), (350, 130)], 8, 8, 256, None),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_values_and_gradients(case):
    seqs, Hq, Hkv, D, room = CASES[case]
    say("cross", case, CASES[case])
    t = cu.Batch(seqs, Hq, Hkv, D, 100 * case + 1, room)
    cu.check(t, cu.run(t), cu.reference(t), "case %d" % case)
