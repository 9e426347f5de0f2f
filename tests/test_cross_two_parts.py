"""Gradients of calls of up to 2^21 scores take P and dS in two bf16 parts, whatever kernel they take: the documented
precision, by the call's own numbers."""
import pytest

import cross_util as cu
import transfer_station_amd as ts

# (B, rows, states, Hq, Hkv, D): up to 2^21 scores, tiles of states few enough and rows many enough that one workgroup's
# eight waves could share a tile
FEW_SCORES = [
    (32, 1, 128, 64, 8, 64),
    (64, 1, 100, 32, 4, 64),
    (8, 1000, 2, 8, 8, 128),
    (4, 2048, 20, 10, 10, 64),
    (2, 2048, 32, 16, 16, 96),
    (1, 8192, 32, 8, 8, 80),  # 2^21
]


@pytest.mark.parametrize("case", range(len(FEW_SCORES)))
def test_kernels_of_two_parts(case):
    B, n, m, Hq, Hkv, D = FEW_SCORES[case]
    assert B * Hq * n * m <= 2 ** 21
    for scores, fine in ((0, True), (1, False)):  # and with bounds of more scores
        claim = m if not scores else 2 ** 21 // (B * Hq * n) + 1
        c = ts.CrossCall(ts.Spans(4096, B * n, n), ts.Spans(4096, B * claim, claim), B, Hq, Hkv, D)
        names = [p[0] for p in ts.attn_cross_plan(c, True) if "_dq_" in p[0] or "_dkv_" in p[0]]
        assert len(names) == 2 and all(x.endswith("true>" if fine else "false>") for x in names), names


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(FEW_SCORES)))
def test_gradients_in_two_parts(case):
    assert ts.device_count() >= 1
    B, n, m, Hq, Hkv, D = FEW_SCORES[case]
    print("two parts", FEW_SCORES[case], flush=True)
    t = cu.Batch([(n, m)] * B, Hq, Hkv, D, 500 + case)
    got = cu.run(t)
    t.fine = (True, True)  # what is documented, not what the plan says
    cu.check(t, got, cu.reference(t), "case %d" % case)
