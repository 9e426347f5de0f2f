"""A launch has less than 2^32 work-items: calls within the documented limits whose tiles, or groups, are more than that."""
import os
import subprocess

import numpy as np
import pytest

import cross_util as cu
import transfer_station_amd as ts

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
CSRC = os.path.join(ROOT, "transfer_station_amd", "csrc")

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


def test_reorder_launches_under_asan_ubsan(tmp_path):
    exe = str(tmp_path / "reorder_checks")
    cmd = ["gcc", "-O1", "-g", "-std=gnu11", "-Wall", "-Wextra", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=all", "-fno-omit-frame-pointer", "-D__HIP_PLATFORM_AMD__=1",
           "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-I" + os.path.join(ROCM, "include"),
           os.path.join(ROOT, "tests", "sanitize", "reorder_checks.c"), os.path.join(CSRC, "attn_beam.c"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    print(r.stdout[-3000:], r.stderr[-3000:])
    assert r.returncode == 0 and "REORDER_CHECKS OK" in r.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("tables", [0, 1])
def test_reorder_of_groups_behind_the_first_launch(tables):
    """2^20 sequences in pairs, 64 or 65 workgroups a pair; a few pairs hold tokens, at the edges of the launches."""
    assert ts.device_count() >= 1
    print("pairs", tables, flush=True)
    B, D, page, n = 1 << 20, 256, 256, 300
    per = (1 << 24) // 64
    pairs = [0, 1, 0xffffff // 65 - 1, 0xffffff // 65, per - 1, per, B // 4, B // 2 - 1]
    rng = np.random.default_rng(3)
    pages = 4 * len(pairs)
    data = {x: rng.integers(0, 256, (pages, page, 2 * D), np.uint8) for x in "kv"}
    table, lens = np.full((B, 2), -1, np.int32), np.zeros(B, np.int32)
    parent = np.arange(B, dtype=np.int32) ^ 1  # every pair changes places
    for i, p in enumerate(pairs):
        lens[2 * p:2 * p + 2] = n
        table[2 * p:2 * p + 2] = 4 * i + np.arange(4).reshape(2, 2)
    want_table, want = table.copy(), {x: a.copy() for x, a in data.items()}
    for p in pairs:
        a, b = table[2 * p], table[2 * p + 1]
        if tables:
            want_table[2 * p, 0], want_table[2 * p + 1, 0] = b[0], a[0]
        for x in "kv":
            want[x][a[1], :n - page], want[x][b[1], :n - page] = data[x][b[1], :n - page], data[x][a[1], :n - page]
    bufs = {x: ts.DeviceBuffer.from_array(a) for x, a in data.items()}
    with ts.DeviceBuffer.from_array(table) as dt, ts.DeviceBuffer.from_array(lens) as dl, \
            ts.DeviceBuffer.from_array(parent) as dp:
        c = ts.KvCache(bufs["k"], bufs["v"], dt, dl, dl, B, 2, pages, page, 1, D, 16)
        ts.attn_kv_reorder(c, dp, 2, tables)
        ts.synchronize()
        assert np.array_equal(dt.download(np.int32).reshape(B, 2), want_table)
    for x, buf in bufs.items():
        assert np.array_equal(buf.download(np.uint8).reshape(want[x].shape), want[x]), x
        buf.free()
