"""CPU tests of cross attention's and beam search's host side: refusals, the choice of kernels, the index arithmetic that
host and kernels share under AddressSanitizer and UndefinedBehaviorSanitizer (tests/sanitize/cross_checks.c), and the
tests' own gradients against differences."""
import os
import re
import signal
import subprocess
import sys

import numpy as np
import pytest

import cross_util as cu
import transfer_station_amd as ts

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
CSRC = os.path.join(ROOT, "transfer_station_amd", "csrc")


def test_index_arithmetic_and_workspaces_under_asan_ubsan(tmp_path):
    exe = str(tmp_path / "cross_checks")
    cmd = ["gcc", "-O1", "-g", "-std=gnu11", "-Wall", "-Wextra", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=all", "-fno-omit-frame-pointer", "-D__HIP_PLATFORM_AMD__=1",
           "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-I" + os.path.join(ROCM, "include"),
           os.path.join(ROOT, "tests", "sanitize", "cross_checks.c"), os.path.join(CSRC, "attn_cross.c"),
           os.path.join(CSRC, "attn_beam.c"), "-lm", "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    print(r.stdout[-3000:], r.stderr[-3000:])
    assert r.returncode == 0 and "CROSS_CHECKS OK" in r.stdout
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr


def test_header_constants():
    text = open(os.path.join(ROOT, "include", "attn_flash.h")).read()
    for k in ("ATTN_TOKEN_MAX", "ATTN_BEAMS_MAX", "ATTN_BEAM_K_MAX", "ATTN_BEAM_V_MAX", "ATTN_REORDER_MAX"):
        assert int(re.search(r"#define %s (\d+)" % k, text).group(1)) == getattr(ts, k)


PRE = """
import transfer_station_amd as ts
def spans(**k):
    a = dict(start=4096, T=100, max=10)
    a.update(k)
    return ts.Spans(**a)
def call(q=None, k=None, **o):
    a = dict(B=2, Hq=8, Hkv=2, D=128)
    a.update(o)
    return ts.CrossCall(q or spans(), k or spans(), **a)
def beams(**k):
    a = dict(logits=4096, row=1000, bits=16, B=2, beams=4, V=1000, K=8, scores=4096)
    a.update(k)
    return ts.Beams(**a)
def cache(**k):
    a = dict(k=4096, v=4096, table=4096, kv_len=4096, q_start=4096, B=8, table_cols=4, pages=8, page=16,
             Hkv=2, D=128, bits=16)
    a.update(k)
    return ts.KvCache(**a)
r, o, x, y, z = (ts.Rows(4096 * i, 1024, 128) for i in range(1, 6))
class none:  # NULL
    _at = None
"""


def cross(c="call()", q="r", k="r", v="r", out="o", lse=4096, s=4096):
    return "ts.attn_cross(%s, %s, %s, %s, %s, %s, %s)" % (c, q, k, v, out, lse, s)


def grad(c="call()", q="r", k="r", v="r", out="o", lse=4096, go="o", dq="x", dk="y", dv="z", s=4096):
    return "ts.attn_cross_grad(%s, %s, %s, %s, %s, %s, %s, %s, %s, %s, %s)" % (c, q, k, v, out, lse, go, dq, dk, dv, s)


def select(c="beams()", score=8192, token=4096 * 4, parent=4096 * 5, s=4096):
    return "ts.attn_beam_select(%s, %s, %s, %s, %s)" % (c, score, token, parent, s)


def reorder(c="cache()", parent=4096, n=4, tables=1):
    return "ts.attn_kv_reorder(%s, %s, %s, %s)" % (c, parent, n, tables)


ROWS = "needs a 16-byte aligned"
SPANS = "needs device pointers to int32"
REFUSED = [
    (cross("none"), "attn_cross: the call must be non-NULL"),
    (cross("call(D=24)"), "D % 16 == 0"),
    (cross("call(D=0)"), "D % 16 == 0"),
    (cross("call(D=272)"), "D % 16 == 0"),
    (cross("call(B=0)"), "need B >= 1"),
    (cross("call(Hkv=0)"), "need B >= 1"),
    (cross("call(Hq=0)"), "need B >= 1"),
    (cross("call(Hq=7)"), "Hq % Hkv"),
    (cross("call(B=2**19, Hkv=4)"), "B * Hkv <= 2^20"),
    (cross("call(spans(start=None))"), "q " + SPANS),
    (cross("call(spans(start=4098))"), "q " + SPANS),
    (cross("call(spans(len=4097))"), "q " + SPANS),
    (cross("call(spans(T=0))"), "q " + SPANS),
    (cross("call(spans(T=2**30 + 1))"), "q " + SPANS),
    (cross("call(spans(max=0))"), "q " + SPANS),
    (cross("call(k=spans(max=-1))"), "k " + SPANS),
    (cross("call(spans(T=2**28), Hq=8)"), "q.T * Hq <= 2^30"),
    (cross("call(k=spans(T=2**30))"), "k.T * Hkv <= 2^30"),
    (cross("call(B=2**18, Hkv=4, k=spans(T=2**22))"), "too many tiles"),
    (cross("call(B=2**16, spans=None)").replace("spans=None", "Hkv=8, q=spans(T=2**24, max=2**24)"), "too many tiles"),
    (cross("call(scale=-1.0)"), "scale must be"),
    (cross("call(scale=float('nan'))"), "scale must be"),
    (cross(q="none"), "q " + ROWS),
    (cross(k="ts.Rows(4104, 1024, 128)"), "k " + ROWS),
    (cross(v="ts.Rows(4096, 1020, 128)"), "v " + ROWS),
    (cross(out="ts.Rows(8192, 1024, 4)"), "o " + ROWS),
    (cross(q="ts.Rows(4096, 120, 128)"), "q " + ROWS),
    (cross(q="ts.Rows(4096, 0, 128)"), "q " + ROWS),
    (cross(k="ts.Rows(4096, 2**22 + 8, 128)"), "k " + ROWS),
    (cross(k="ts.Rows(4096, 1024, -128)"), "k " + ROWS),
    (cross(out="r"), "o must not be q, k or v"),
    (cross(out="ts.Rows(8192, 1024, 64)"), "heads of o must not overlap"),
    (grad(dq="ts.Rows(4096 * 9, 1024, 0)"), "heads of dq must not overlap"),
    (grad(dv="ts.Rows(4096 * 9, 1024, 120)"), "heads of dv must not overlap"),
    (cross(lse=4097), "lse must be"),
    (cross(s="None"), "scratch must be"),
    (cross(s=4128), "scratch must be"),
    (grad("none"), "attn_cross_grad: the call must be non-NULL"),
    (grad(go="none"), "d_o " + ROWS),
    (grad(dq="ts.Rows(None, 1024, 128)"), "dq " + ROWS),
    (grad(dk="ts.Rows(4096 * 7, 64, 128)"), "dk " + ROWS),
    (grad(dv="none"), "dv " + ROWS),
    (grad(dq="r"), "dq, dk and dv must be none"),
    (grad(dk="o"), "dq, dk and dv must be none"),
    (grad(dv="y"), "dq, dk and dv must be none"),
    (grad(lse="None"), "lse must be"),
    (grad(s=32), "scratch must be"),
    ("ts.attn_cross_scratch_bytes(call(D=8))", "attn_cross_scratch_bytes: need D"),
    ("ts.attn_cross_grad_scratch_bytes(call(B=-1))", "attn_cross_grad_scratch_bytes: need B"),
    ("ts.attn_cross_plan(call(Hq=5))", "attn_cross_plan: need B"),
    (select("none"), "attn_beam_select: the beams must be non-NULL"),
    (select("beams(bits=8)"), "bits must be 16"),
    (select("beams(B=0)"), "need B >= 1"),
    (select("beams(beams=0)"), "beams in [1, 256]"),
    (select("beams(beams=257)"), "beams in [1, 256]"),
    (select("beams(K=0)"), "K in [1, 64]"),
    (select("beams(K=65)"), "K in [1, 64]"),
    (select("beams(V=0)"), "V in [1, 2^20]"),
    (select("beams(V=2**20 + 1, row=2**21)"), "V in [1, 2^20]"),
    (select("beams(B=2**13, beams=256)"), "B * beams <= 2^20"),
    (select("beams(row=999)"), "row at least V"),
    (select("beams(logits=4097)"), "aligned to its elements"),
    (select("beams(logits=4098, bits=32)"), "aligned to its elements"),
    (select("beams(scores=None)"), "scores must be"),
    (select("beams(done=4096, done_token=1000)"), "done_token must be"),
    (select("beams(done=4096, done_token=-1)"), "done_token must be"),
    (select(score=4096), "must be four arrays"),
    (select(token=4096 * 3, parent=4096 * 3), "must be four arrays"),
    (select(token=8192), "must be four arrays"),
    (select(token="None"), "score, token and parent"),
    (select(parent=4098), "score, token and parent"),
    (select(s=16), "scratch must be"),
    ("ts.attn_beam_scratch_bytes(beams(K=100))", "attn_beam_scratch_bytes: need B"),
    (reorder("none"), "attn_kv_reorder: the cache must be non-NULL"),
    (reorder("cache(bits=8)"), "bits must be"),
    (reorder("cache(D=40)"), "a bf16 cache needs"),
    (reorder("cache(D=96, bits=4, k_scale=4096, v_scale=4096)"), "a 4-bit one D of"),
    (reorder("cache(page=24)"), "page must be"),
    (reorder("cache(B=0)"), "need B, Hkv"),
    (reorder("cache(table_cols=2**27)"), "rows of 2^30 tokens"),
    (reorder(n=0), "beams in [1, 32]"),
    (reorder(n=33), "beams in [1, 32]"),
    (reorder(n=3), "B % beams == 0"),
    (reorder("cache(k=None)"), "k and v"),
    (reorder("cache(bits=4)"), "k and v"),
    (reorder("cache(table=None)"), "table, kv_len and parent"),
    (reorder(parent="None"), "table, kv_len and parent"),
    (reorder("cache(Hkv=2**16, page=256)"), "2^29 elements"),
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
    # grad, D, B, Hq, Hkv, max q, max k, the kernels, in order: name, notes, grid
    # few rows: shares of 256 workgroups, or whole sequences where those are enough and short
    (0, 64, 1, 16, 16, 1, 1500, [("rows_kernel<64, 1, true, 4>", "parts=64 share=1", 192), ("merge_kernel<16, 1>", "", 1)]),
    (0, 64, 16, 16, 16, 5, 1500, [("rows_kernel<64, 1, true, 4>", "parts=1 share=1", 256)]),
    (0, 128, 1, 32, 8, 1, 32768, [("rows_kernel<128, 1, true, 4>", "parts=64 share=1", 256), ("merge_kernel<16, 4>", "", 16)]),
    # much to read of four kv heads and more: a wave each
    (0, 128, 64, 32, 8, 1, 8192, [("rows_kernel<128, 1, true, 1>", "parts=32 share=1", 256), ("merge_kernel<4, 1>", "", 256)]),
    (0, 128, 64, 24, 6, 1, 8192, [("rows_kernel<128, 1, true, 4>", "parts=42 share=1", 256), ("merge_kernel<4, 1>", "", 192)]),
    # two blocks of 16 rows, past D = 128 one, twice
    (0, 128, 4, 32, 8, 8, 3000, [("rows_kernel<128, 2, true, 4>", "parts=64 share=1", 256), ("merge_kernel<16, 1>", "", 128)]),
    (0, 256, 4, 32, 8, 8, 3000, [("rows_kernel<256, 1, false, 4>", "parts=64 share=1", 256), ("merge_kernel<16, 1>", "", 256)]),
    # more rows: tiles of 128, in parts where they are few
    (0, 128, 1, 32, 8, 9, 3000, [("kernel<128>", "parts=11 share=384", 88), ("merge_kernel<16, 1>", "", 36)]),
    (0, 80, 8, 16, 16, 1000, 1500, [("kernel<96>", "parts=1 share=1536", 1024)]),
    (0, 112, 8, 16, 16, 1000, 1500, [("kernel<128>", "parts=1 share=1536", 1024)]),
    # rows for too many partial slots: no parts
    (0, 64, 70000, 1, 1, 1, 2, [("rows_kernel<64, 1, true, 4>", "parts=1 share=1", 70000)]),
    (1, 64, 3, 8, 8, 37, 50, [("dq_kernel<64, true>", "parts=1 share=128", 24),
                              ("dkv_kernel<64, true, true, 1, true>", "parts=1 share=2", 24)]),
    # up to 2^21 scores P and dS in two parts
    (1, 64, 1, 4, 4, 1024, 512, [("dq_kernel<64, true>", "parts=2 share=256", 64), ("sum_kernel<false>", "", 256),
                                 ("dkv_kernel<64, true, true, 1, true>", "parts=16 share=2", 256), ("sum_kernel<true>", "", 256)]),
    (1, 64, 1, 4, 4, 1024, 513, [("dq_kernel<64, false>", "parts=2 share=384", 64), ("sum_kernel<false>", "", 256),
                                 ("dkv_kernel<64, true, true, 1, false>", "parts=16 share=2", 320), ("sum_kernel<true>", "", 257)]),
    (1, 64, 4, 10, 10, 4096, 77, [("dq_kernel<64, false>", "parts=1 share=128", 1280),
                                  ("dkv_kernel<64, true, true, 2, false>", "parts=6 share=22", 240), ("sum_kernel<true>", "", 388)]),
    (1, 128, 2, 32, 8, 4096, 4096, [("dq_kernel<128, false>", "parts=1 share=4096", 2048),
                                    ("dkv_kernel<128, true, true, 1, false>", "parts=1 share=512", 512)]),
    (1, 256, 1, 4, 2, 100, 9000, [("dq_kernel<256, false>", "parts=35 share=384", 140), ("sum_kernel<false>", "", 100),
                                  ("dkv_kernel<256, true, false, 1, false>", "parts=1 share=8", 142),
                                  ("dkv_kernel<256, false, true, 1, false>", "parts=1 share=8", 142)]),
]


@pytest.mark.parametrize("case", range(len(PLANS)))
def test_kernel_choice(case):
    """The cut at both sides of its rules: it goes by the call's numbers alone."""
    g, D, B, Hq, Hkv, mq, mk, want = PLANS[case]
    c = ts.CrossCall(ts.Spans(4096, B * mq, mq), ts.Spans(4096, B * mk, mk), B, Hq, Hkv, D)
    p = ts.attn_cross_plan(c, g)
    print(p)
    got = [(n.replace("attn_cross_", ""), notes, int(grid)) for n, notes, grid, _ in p]
    assert [(n, x) for n, _, x in got] == [(n, x) for n, _, x in want]
    assert all(a[1] == b[1] for a, b in zip(got, want))


def test_scores_past_64_bits():
    """8 sequences that may each have 2^30 rows and 2^30 states: 2^63 scores are not few."""
    c = ts.CrossCall(ts.Spans(4096, 2 ** 30, 2 ** 30), ts.Spans(4096, 2 ** 30, 2 ** 30), 8, 1, 1, 64)
    names = [p[0] for p in ts.attn_cross_plan(c, True) if "sum" not in p[0]]
    assert names and all(n.endswith("false>") for n in names), names


def test_bounds_past_the_tensor_are_cut():
    """max above T asks for no more workgroups than T rows need."""
    def plan(mq, mk):
        return ts.attn_cross_plan(ts.CrossCall(ts.Spans(4096, 300, mq), ts.Spans(4096, 500, mk), 1, 8, 8, 64))

    assert plan(300, 500) == plan(2 ** 31 - 1, 2 ** 31 - 1)


def test_gradients_of_the_reference_by_differences():
    """The tests' dq, dk and dv against central differences of sum(dO o O), in float64."""
    t = cu.Batch([(3, 5), (4, 2), (2, 0)], 4, 2, 16, 5)
    ref = cu.reference(t)
    rng = np.random.default_rng(0)

    def value():
        out = 0.0
        for b, (n, m) in enumerate(t.seqs):
            rows, states = t.rows(b)
            if not m:
                continue
            for h in range(t.Hq):
                Q, K, V, G = (X[x][r, i] for x, r, i in (("q", rows, h), ("k", states, h // 2), ("v", states, h // 2),
                                                         ("go", rows, h)))
                S = Q @ K.T * t.D ** -0.5
                w = np.exp(S - S.max(1, keepdims=True))
                out += np.sum(G * ((w / w.sum(1, keepdims=True)) @ V))
        return out

    X = {}
    for x, heads in (("q", t.Hq), ("go", t.Hq), ("k", t.Hkv), ("v", t.Hkv)):
        live = t.live_q if heads == t.Hq else t.live_k
        a = cu.f32(np.where(live[:, None], getattr(t, x), 0)[:, :heads * t.D]).astype(np.float64)
        X[x] = a.reshape(-1, heads, t.D)
    for x, d in (("q", "dq"), ("k", "dk"), ("v", "dv")):
        step = rng.standard_normal(X[x].shape)
        base = X[x]
        X[x] = base + 1e-5 * step
        hi = value()
        X[x] = base - 1e-5 * step
        lo = value()
        X[x] = base
        # The third derivative's share of a step of 1e-5 is 1e-10 of the value, and so is cancellation's.
        assert abs((hi - lo) / 2e-5 - np.sum(ref[d][0] * step)) < 1e-7 * max(1.0, abs(hi))
