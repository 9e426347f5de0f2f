"""A launch has less than 2^32 work-items: calls within the documented limits whose tiles are more than that."""
import numpy as np
import pytest

import cross_util as cu
import transfer_station_amd as ts

# (B, Hq, Hkv, D, q.T, q.max, k.T, k.max): 2^33 work-items and more for a workgroup of 256 threads per tile
WIDE = [
    (4096, 8, 8, 64, 1 << 17, 1 << 17, 1 << 15, 64),             # 2^25 tiles of rows
    (1 << 20, 1, 1, 16, 16256, 16256, 50, 50),                   # 127 tiles of rows of 2^20 sequences
    (1 << 19, 2, 2, 128, 900, 900, 130048, 130048),              # 1016 tiles of states of 2^20 sequences and heads
    (4096, 64, 4, 80, 65408, 65408, 1 << 18, 1 << 18),           # both
    (16384, 1, 1, 256, 1 << 19, 2 ** 31 - 1, 1 << 20, 1 << 20),
]


@pytest.mark.parametrize("case", range(len(WIDE)))
@pytest.mark.parametrize("grad", [False, True])
def test_work_items_of_every_launch(case, grad):
    B, Hq, Hkv, D, qT, qm, kT, km = WIDE[case]
    c = ts.CrossCall(ts.Spans(4096, qT, qm), ts.Spans(4096, kT, km), B, Hq, Hkv, D)
    plan = ts.attn_cross_plan(c, grad)
    print(plan)
    assert plan
    for name, _, grid, block in plan:
        assert 0 < int(grid) * int(block) < 2 ** 32, (name, grid, block)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,states", [(140000, 40), (40, 140000)])
def test_tiles_that_no_workgroup_is_launched_for(rows, states):
    """16384 sequences that may each have over 2^18 rows, or states: the one that has as many takes second turns."""
    assert ts.device_count() >= 1
    print("wide", rows, states, flush=True)
    seqs = [(0, 0)] * 16384
    seqs[0], seqs[9000], seqs[16383] = (34, 70), (rows, states), (130, 33)
    t = cu.Batch(seqs, 1, 1, 16, 31, pad=130000)
    got = cu.run(t, max_q=max(rows, 34), max_k=max(states, 70))
    cu.check(t, got, cu.reference(t))
