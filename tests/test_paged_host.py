"""CPU tests of the paged cache's host side: its refusals, its constants, and, under AddressSanitizer and
UndefinedBehaviorSanitizer, the index arithmetic that host and kernels share (tests/sanitize/paged_checks.c)."""
import os
import re
import signal
import subprocess
import sys

import numpy as np
import pytest

import paged_util as pu
import transfer_station_amd as ts

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


def test_index_arithmetic_under_asan_ubsan(tmp_path):
    exe = str(tmp_path / "paged_checks")
    cmd = ["gcc", "-O1", "-g", "-std=gnu11", "-Wall", "-Wextra", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=all", "-fno-omit-frame-pointer", "-D__HIP_PLATFORM_AMD__=1",
           "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "transfer_station_amd", "csrc"),
           "-I" + os.path.join(ROCM, "include"), os.path.join(ROOT, "tests", "sanitize", "paged_checks.c"),
           os.path.join(ROOT, "transfer_station_amd", "csrc", "attn_paged.c"), "-lm", "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    print(r.stdout[-3000:], r.stderr[-3000:])
    assert r.returncode == 0 and "PAGED_CHECKS OK" in r.stdout
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr


def test_header_constants():
    text = open(os.path.join(ROOT, "include", "attn_flash.h")).read()
    for k in ("ATTN_KV_BF16", "ATTN_KV_FP4", "ATTN_KV_PAGE_MIN", "ATTN_KV_PAGE_MAX"):
        assert int(re.search(r"#define %s (\d+)" % k, text).group(1)) == getattr(ts, k)


PRE = """
import transfer_station_amd as ts
def cache(**k):
    a = dict(k=4096, v=4096, table=4096, kv_len=4096, q_start=4096, B=2, table_cols=4, pages=8, page=16,
             Hkv=2, D=128, bits=16)
    a.update(k)
    return ts.KvCache(**a)
r = ts.Rows(4096, 1024, 128)
class none:  # NULL
    _at = None
"""
FOUR = "bits=4, k_scale=4096, v_scale=4096"
ATTEND = "ts.attn_paged(%s, %s, %s, %s, %s, 1, %s, %s, %s, %s)"


def attend(c="cache()", q="r", o="r", T=4, Hq=8, sc="None", mq=1, mk=64, s=4096):
    return ATTEND % (c, q, o, T, Hq, sc, mq, mk, s)


APPEND = "ts.attn_kv_append(%s, %s, %s, %s, %s, %s, %s, %s, %s, %s, 0, %s)"


def append(c="cache()", q="r", qo="r", k="r", v="r", T=4, Hq=8, rope=4096, rows=64, rot=128, mq=1):
    return APPEND % (c, q, qo, k, v, T, Hq, rope, rows, rot, mq)


REFUSED = [
    (attend("none"), "attn_paged: the cache must be non-NULL"),
    (attend("cache(bits=8)"), "bits must be"),
    (attend("cache(D=24)"), "D % 16 == 0"),
    (attend("cache(D=0)"), "D % 16 == 0"),
    (attend("cache(D=272)"), "D % 16 == 0"),
    (attend("cache(D=96, %s)" % FOUR), "D of 64, 128 or 256"),
    (attend("cache(page=8)"), "power of two in [16, 256]"),
    (attend("cache(page=48)"), "power of two in [16, 256]"),
    (attend("cache(page=512)"), "power of two in [16, 256]"),
    (attend("cache(B=0)"), "need B >= 1"),
    (attend("cache(Hkv=0)"), "need B >= 1"),
    (attend("cache(pages=0)"), "need B >= 1"),
    (attend("cache(table_cols=0)"), "need B >= 1"),
    (attend("cache(table_cols=2**27)"), "at most 2^30 tokens"),
    (attend("cache(B=2**10, table_cols=2**25, Hkv=2**10)"), "at most 2^38 tokens"),
    (attend("cache(k=None)"), "k and v must be"),
    (attend("cache(v=4104)"), "k and v must be"),
    (attend("cache(bits=4)"), "k_scale and v_scale"),
    (attend("cache(bits=4, k_scale=4096, v_scale=4097)"), "k_scale and v_scale"),
    (attend("cache(table=None)"), "table, kv_len and q_start"),
    (attend("cache(kv_len=4098)"), "table, kv_len and q_start"),
    (attend("cache(q_start=None)"), "table, kv_len and q_start"),
    (attend(T=0), "need T in"),
    (attend(T=2 ** 30 + 1), "need T in"),
    (attend(Hq=0), "Hq % Hkv"),
    (attend(Hq=3), "Hq % Hkv"),
    (attend(T=2 ** 28, Hq=8), "T * Hq <= 2^30"),
    (attend(mq=0), "max_q >= 1"),
    (attend(mk=0), "max_kv >= 1"),
    (attend(q="none"), "q needs a 16-byte aligned"),
    (attend(q="ts.Rows(4100, 1024, 128)"), "q needs a 16-byte aligned"),
    (attend(o="ts.Rows(4096, 1020, 128)"), "o needs a 16-byte aligned"),
    (attend(o="ts.Rows(4096, 1024, -128)"), "o needs a 16-byte aligned"),
    (attend(o="ts.Rows(None, 1024, 128)"), "o needs a 16-byte aligned"),
    (attend(sc="ts.Scores(-1.0)"), "scale must be"),
    (attend(sc="ts.Scores(float('nan'))"), "scale must be"),
    (attend(sc="ts.Scores(0.0, -2.0)"), "softcap must be"),
    (attend(sc="ts.Scores(0.0, float('inf'))"), "softcap must be"),
    (attend(sc="ts.Scores(0.0, 0.0, 4097)"), "slopes must be"),
    (attend(s="None"), "scratch must be"),
    (attend(s=4128), "scratch must be"),
    (attend(), "o must not be q"),
    (append("none"), "attn_kv_append: the cache must be non-NULL"),
    (append(Hq=5), "Hq % Hkv"),
    (append(q="None"), "q_out without q"),
    (append(qo="None"), "q_out needs"),
    (append(qo="ts.Rows(r.data, r.token + 8, r.head)"), "needs q's strides"),
    (append(qo="ts.Rows(r.data, r.token, r.head + 8)"), "needs q's strides"),
    (append(k="none"), "k needs"),
    (append(v="ts.Rows(4096, 4, 8)"), "v needs"),
    (append(rot=136), "rot must be"),
    (append(rot=144), "rot must be"),
    (append(rot=-16), "rot must be"),
    (append(rope="None"), "rope must be"),
    (append(rope=4100), "rope must be"),
    (append(rows=0), "rope must be"),
    (append(mq=0), "max_q >= 1"),
    (attend("cache(B=2**17, Hkv=16)"), "B * Hkv <= 2^20"),
    ("ts.attn_kv_read(cache(D=40), r, r, 4, 1)", "attn_kv_read: a bf16 cache"),
    ("ts.attn_kv_read(cache(), none, r, 4, 1)", "k needs"),
    ("ts.attn_kv_read(cache(), r, ts.Rows(4096, 8, 9), 4, 1)", "v needs"),
    ("ts.attn_kv_read(cache(), r, r, 4, 0)", "max_q >= 1"),
    ("ts.attn_paged_plan(cache(page=20), 4, 8, 1, None, 1, 1)", "attn_paged_plan: page must be"),
]


def test_refusals():
    """Each ends its process with a message before any device call; run side by side."""
    def start(code):
        return subprocess.Popen([sys.executable, "-c", "import sys; sys.path.insert(0, %r)\n" % ROOT + PRE + code],
                                stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)

    for i in range(0, len(REFUSED), 8):
        procs = [(c, m, start(c)) for c, m in REFUSED[i:i + 8]]
        for code, msg, p in procs:
            err = p.communicate(timeout=120)[1]
            assert p.returncode == -signal.SIGABRT, (code, err)
            assert msg in err, (code, err)


PLANS = [
    # bits, D, B, Hq, Hkv, max_q, max_kv, causal, modified scores, first kernel, its notes, grid, kernels
    # one to 16 rows of a kv head: 512 workgroups, 256 in bf16 past D = 128, fewer where there are fewer units
    (16, 128, 64, 32, 8, 1, 8192, 1, 0, "decode_kernel<128, 16, 1, false, true>", "teams=512 parts=32", 512, 2),
    (16, 128, 1, 32, 8, 1, 777, 1, 0, "decode_kernel<128, 16, 1, false, true>", "teams=56 parts=8", 56, 2),
    (16, 256, 32, 32, 8, 1, 4096, 1, 0, "decode_kernel<256, 16, 1, false, true>", "teams=256 parts=33", 256, 2),
    (4, 256, 32, 32, 8, 1, 4096, 1, 1, "decode_kernel<256, 4, 1, true, true>", "teams=512 parts=33", 512, 2),
    (4, 256, 1, 16, 4, 1, 32768, 1, 0, "decode_kernel<256, 4, 1, false, true>", "teams=256 parts=256", 256, 2),
    # more rows in all than there are partial slots for two parts: a workgroup per sequence
    (16, 64, 2100, 32, 8, 1, 500, 1, 0, "decode_kernel<64, 16, 1, false, true>", "teams=0 parts=1", 16800, 1),
    # two row blocks; at D > 128 one, twice
    (16, 128, 16, 32, 8, 8, 4000, 1, 0, "decode_kernel<128, 16, 2, false, true>", "teams=512 parts=16", 512, 2),
    (4, 256, 16, 32, 8, 8, 4000, 1, 0, "decode_kernel<256, 4, 1, false, false>", "teams=256 parts=16", 512, 2),
    # 33 to 64 rows: key halves of four waves
    (16, 128, 16, 64, 8, 8, 4001, 1, 1, "prefill_kernel<128, 16, true, 2, 4>", "parts=4 share=1024", 512, 2),
    (16, 256, 16, 64, 8, 8, 4001, 1, 0, "decode_kernel<256, 16, 1, false, false>", "teams=64 parts=8", 256, 2),
    # more: up to a round of tiles, and two of a causal prompt, on key halves of eight waves
    (16, 128, 1, 32, 8, 512, 8192, 1, 0, "prefill_kernel<128, 16, false, 2, 8>", "parts=2 share=4096", 256, 2),
    (16, 128, 1, 32, 8, 1024, 8192, 1, 0, "prefill_kernel<128, 16, false, 2, 8>", "parts=1 share=1073741824", 256, 1),
    (16, 128, 1, 32, 8, 2048, 2048, 1, 0, "prefill_kernel<128, 16, false, 2, 8>", "parts=1 share=1073741824", 512, 1),
    (16, 128, 1, 32, 8, 2048, 2048, 0, 0, "prefill_kernel<128, 16, false, 1, 4>", "parts=1 share=1073741824", 512, 1),
    (16, 128, 1, 32, 8, 1200, 8192, 1, 0, "prefill_kernel<128, 16, false, 1, 4>", "parts=1 share=1073741824", 304, 1),
    (4, 64, 6, 24, 6, 2000, 3000, 1, 0, "prefill_kernel<64, 4, false, 1, 4>", "parts=1 share=1073741824", 2304, 1),
    (16, 256, 1, 32, 8, 512, 4096, 1, 0, "prefill_kernel<256, 16, false, 1, 4>", "parts=4 share=1024", 512, 2),
]


@pytest.mark.parametrize("case", PLANS, ids=[str(i) for i in range(len(PLANS))])
def test_kernel_choice(case):
    """The cut at both sides of its rules: it goes by the call's numbers alone."""
    bits, D, B, Hq, Hkv, mq, mk, causal, mod, name, notes, grid, n = case
    c = ts.KvCache(4096, 4096, 4096, 4096, 4096, B, 65536 // 64, 1000, 64, Hkv, D, bits, 4096, 4096)
    p = ts.attn_paged_plan(c, B * mq, Hq, causal, ts.Scores(0.0, 30.0 if mod else 0.0), mq, mk)
    print(p)
    assert p[0][0] == "attn_paged_" + name and p[0][1] == notes and int(p[0][2]) == grid
    assert len(p) == n and (n == 1 or p[1][0].startswith("attn_paged_merge_kernel<"))


def test_reference_quantiser():
    """The tests' own quantiser against the definition, element by element."""
    x = pu.normal((4, 64), 3, 5.0)
    x[0, :32] = 0
    x[1, :4] = pu.bf16(np.array([7.0, 5.0, 2.5, -3.5], np.float32))
    x[1, 4:32] = 0
    codes, scales = pu.quantise(x)
    v = pu.values4(codes, scales)
    assert np.all(v[0, :32] == 0) and np.array_equal(v[1, :4], [6, 4, 2, -4])
    f = pu.f32(x).astype(np.float64)
    for r in range(4):
        for gr in range(2):
            a, s = np.abs(f[r, 32 * gr:32 * gr + 32]), 2.0 ** (int(scales[r, gr]) - 127)
            assert a.max() <= 7 * s and (a.max() == 0 or a.max() > 3.5 * s)
            d = np.abs(a[:, None] / s - pu.LEVELS).min(1)
            got = np.abs(a / s - np.abs(v[r, 32 * gr:32 * gr + 32]) / s)
            assert np.allclose(got, d, rtol=0, atol=1e-12)
