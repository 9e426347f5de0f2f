"""The paged KV cache on the GPU: append, read back and attention against numpy, in bf16 and in 4 bits. What no
token fills in the cache, the scratch and the outputs start as NaN."""
import numpy as np
import pytest

import paged_util as pu
import transfer_station_amd as ts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu_present():
    assert ts.device_count() >= 1, "no HIP device visible: GPU tests must run on the MI355X box"


def check(O, ref, bound, what):
    assert np.all(np.isfinite(O)), what
    off = np.abs(O - ref) - bound
    assert off.max(initial=0.0) <= 0.0, (what, float(off.max()), np.unravel_index(off.argmax(), off.shape))


# ---- append and read -------------------------------------------------------------------------
def append(cache, qkv, Hq, rope, rot, pairs, max_q=None, in_place=False, with_q=True, pad=2):
    """qkv [N][Hq + 2 Hkv][D] bf16 in one padded tensor; returns q_out [N][Hq][D]."""
    N, H, D = qkv.shape
    T, Hkv = N + pad, cache.Hkv
    full = np.full((T, H, D), 0xFFFF, np.uint16)
    full[:N] = qkv
    desc = cache.device()
    with ts.DeviceBuffer.from_array(full) as dx, ts.DeviceBuffer(T * Hq * D * 2) as dq, \
            ts.DeviceBuffer.from_array(rope) as dr:
        dq.fill_bytes(0xFF)
        q = ts.Rows(dx, H * D, D)
        out = q if in_place else ts.Rows(dq, Hq * D, D)
        k = ts.Rows(dx.ptr + 2 * Hq * D, H * D, D)
        v = ts.Rows(dx.ptr + 2 * (Hq + Hkv) * D, H * D, D)
        ts.attn_kv_append(desc, q if with_q else None, out if with_q else None, k, v, T, Hq, dr,
                          len(rope), rot, pairs, max_q or max(n for n, _ in cache.seqs))
        ts.synchronize()
        got = dx.download(np.uint16).reshape(T, H, D)[:, :Hq] if in_place else \
            dq.download(np.uint16).reshape(T, Hq, D)
    cache.download()
    assert np.all(got[N:] == 0xFFFF)
    return got[:N]


APPEND = [
    # bits, D, page, Hq, Hkv, (new, length) by sequence, rot, pairs, max_q
    (16, 128, 16, 8, 2, [(1, 1)], 128, 0, None),
    (16, 128, 64, 32, 8, [(1, 777), (1, 1), (1, 64), (1, 65)], 128, 0, None),
    (16, 80, 32, 6, 3, [(33, 40), (0, 17), (7, 7)], 32, 0, None),
    (16, 48, 16, 3, 1, [(5, 21), (100, 130)], 48, 1, 3),          # more tokens than max_q says
    (16, 256, 128, 4, 4, [(20, 20)], 0, 0, None),
    (16, 16, 256, 2, 1, [(300, 600)], 16, 1, None),
    (4, 128, 16, 8, 2, [(1, 1), (1, 40)], 128, 0, None),
    (4, 64, 32, 12, 4, [(31, 63), (2, 2)], 32, 1, None),
    (4, 256, 64, 5, 5, [(70, 200), (1, 9)], 256, 1, 8),
    (4, 128, 128, 3, 1, [(9, 130)], 16, 0, None),                 # halves inside one group
    (4, 64, 16, 7, 7, [(3, 3)], 0, 0, None),
]


@pytest.mark.parametrize("case", APPEND, ids=[str(c[:5]) + str(c[6:8]) for c in APPEND])
def test_append_and_read(case):
    """Bit for bit: rotation, rounding and quantisation are defined to the last bit."""
    bits, D, page, Hq, Hkv, seqs, rot, pairs, max_q = case
    print("append", case, flush=True)
    want, got = (pu.Cache(seqs, Hkv, D, page, bits, 5) for _ in range(2))
    want.fill(11)
    got.fill(11)
    qkv = pu.normal((got.N, Hq + 2 * Hkv, D), 77)
    rope = pu.rope_table(max(k for _, k in seqs), rot)
    q = append(got, qkv, Hq, rope, rot, pairs, max_q)
    wq = np.empty((want.N, Hq, D), np.uint16)
    for b, (n, kv) in enumerate(seqs):
        r = slice(want.start[b], want.start[b + 1])
        pos = np.arange(kv - n, kv)
        wq[r] = pu.rotate(qkv[r, :Hq], pos, rope, rot, pairs)
        want.put(b, kv - n, pu.rotate(qkv[r, Hq:Hq + Hkv], pos, rope, rot, pairs), qkv[r, Hq + Hkv:])
    assert np.array_equal(q, wq)
    for x in ("k", "v") + (("ks", "vs") if bits == 4 else ()):
        assert np.array_equal(getattr(got, x), getattr(want, x)), x
    # and back, with the dense layout [heads][tokens][D]
    T = got.N + 1
    with ts.DeviceBuffer(T * Hkv * D * 2) as dk, ts.DeviceBuffer(T * Hkv * D * 2) as dv:
        dk.fill_bytes(0xFF)
        dv.fill_bytes(0xFF)
        ts.attn_kv_read(got.device(), ts.Rows(dk, D, T * D), ts.Rows(dv, D, T * D), T,
                        max_q or max(n for n, _ in seqs))
        ts.synchronize()
        back = [d.download(np.uint16).reshape(Hkv, T, D) for d in (dk, dv)]
    for i, x in enumerate(back):
        assert np.all(x[:, got.N:] == 0xFFFF)
        for b, (n, kv) in enumerate(seqs):
            rows = pu.f32(x[:, got.start[b]:got.start[b + 1]]).astype(np.float64)
            assert np.array_equal(rows.transpose(1, 0, 2), want.get(b, kv - n, kv)[i])


def test_append_in_place_and_without_q():
    seqs, D = [(5, 9), (1, 30)], 128
    rope = pu.rope_table(40, D)
    outs = []
    for in_place, with_q in ((False, True), (True, True), (False, False)):
        c = pu.Cache(seqs, 2, D, 16, 16, 5)
        qkv = pu.normal((c.N, 8, D), 3)
        outs.append((append(c, qkv, 4, rope, D, 0, in_place=in_place, with_q=with_q), c.k, c.v))
    assert np.array_equal(outs[0][0], outs[1][0])
    assert np.all(outs[2][0] == 0xFFFF)
    for o in outs[1:]:
        assert np.array_equal(outs[0][1], o[1]) and np.array_equal(outs[0][2], o[2])


@pytest.mark.parametrize("bits", [16, 4])
def test_append_skips_what_has_no_place(bits):
    """Pages that are none, positions below 0 and past the rope table, lengths past the table's row."""
    D, Hkv, Hq, page = 128, 2, 2, 16
    seqs = [(20, 40), (4, 2), (3, 33), (20, 60), (2, -5)]
    c = pu.Cache(seqs, Hkv, D, page, bits, 9, cols=3)
    c.table[0, 2] = c.pages        # tokens 32 .. 39 of sequence 0: no page
    c.table[2, 2] = -7
    before = [getattr(c, x).copy() for x in ("k", "v", "ks", "vs")]
    qkv = pu.normal((c.N, Hq + 2 * Hkv, D), 21)
    rope = pu.rope_table(46, D)     # sequence 3 covers positions 40 .. 59 of a row of 48
    q = append(c, qkv, Hq, rope, D, 0)
    want = pu.Cache(seqs, Hkv, D, page, bits, 9, cols=3)
    want.table = c.table.copy()
    for b, (n, kv) in enumerate(seqs):
        for i in range(n):
            p, r = kv - n + i, want.start[b] + i
            if 0 <= p < 46:
                assert np.array_equal(q[r:r + 1], pu.rotate(qkv[r:r + 1, :Hq], np.array([p]), rope, D, 0))
            else:
                assert np.all(q[r] == 0xFFFF)
            if 0 <= p < 46 and 0 <= want.table[b, p // page] < want.pages:
                want.put(b, p, pu.rotate(qkv[r:r + 1, Hq:Hq + Hkv], np.array([p]), rope, D, 0),
                         qkv[r:r + 1, Hq + Hkv:])
    for x, old in zip(("k", "v", "ks", "vs"), before):
        assert np.array_equal(getattr(c, x), getattr(want, x)), x
        assert bits == 16 and x in ("ks", "vs") or not np.array_equal(getattr(c, x), old), x
    # read back: zeros where a token has no place
    T = c.N
    with ts.DeviceBuffer(T * Hkv * D * 2) as dk, ts.DeviceBuffer(T * Hkv * D * 2) as dv:
        ts.attn_kv_read(c.device(), ts.Rows(dk, Hkv * D, D), ts.Rows(dv, Hkv * D, D), T, 20)
        ts.synchronize()
        k = dk.download(np.uint16).reshape(T, Hkv, D)
    assert np.all(k[12:20] == 0) and np.all(k[c.start[1]:c.start[1] + 2] == 0)
    assert np.all(k[c.start[3] + 8:c.start[4]] == 0) and np.all(k[c.start[4]:] == 0)


def test_quantiser_over_every_bf16_value():
    """Each finite bf16 value, alone in its group and beside larger ones; a group with a NaN or an infinity
    reads as NaN, its neighbours as before."""
    D, Hkv = 128, 8
    every = np.arange(65536, dtype=np.uint16)
    every = every[np.isfinite(pu.f32(every))]
    rows = [every]
    for up in (1, 2, 3, 4):  # the group's largest element is `up` exponents above
        top = np.minimum(np.abs(pu.f32(every)).astype(np.float64) * 2.0 ** up * 1.3, 3e38)
        rows.append(pu.bf16(top))
    n = -(-len(every) // (D * Hkv // 8))
    flat = np.zeros((n * (D * Hkv // 8), 8), np.uint16)
    flat[:len(every), 0] = every
    for i in range(1, 5):
        flat[:len(every), i] = rows[i]
    flat[::3, 1:] = 0          # every third value (and its successors) alone
    flat[1::3, 2:] = 0
    x = flat.reshape(-1, 32)   # groups of four values with their neighbours
    x = np.concatenate([x, flat[:, 0].reshape(-1, 32)])[:, :]
    pad = -len(x) % (Hkv * D // 32)
    x = np.concatenate([x, np.zeros((pad, 32), np.uint16)]).reshape(-1, Hkv, D)
    bad = x[-4:].copy()
    bad[0, 0, 5], bad[1, 1, 40], bad[2, 2, 127] = 0x7F80, 0xFFC0, 0xFF80
    x = np.concatenate([x, bad])
    N = len(x)
    c = pu.Cache([(N, N)], Hkv, D, 256, 4, 1)
    qkv = np.concatenate([x, x], 1)
    append(c, qkv, 0, np.zeros((1, 1), np.float32), 0, 0, with_q=False)
    codes, scales = pu.quantise(x)
    pg, at = c.places(0, 0, N)
    for got, sc in ((c.k, c.ks), (c.v, c.vs)):
        assert np.array_equal(sc[pg, :, at], scales)
        assert np.array_equal(got[pg, :, at], codes)
    with ts.DeviceBuffer(N * Hkv * D * 2) as dk, ts.DeviceBuffer(N * Hkv * D * 2) as dv:
        ts.attn_kv_read(c.device(), ts.Rows(dk, Hkv * D, D), ts.Rows(dv, Hkv * D, D), N, N)
        ts.synchronize()
        k = pu.f32(dk.download(np.uint16)).reshape(x.shape)
    want = pu.values4(codes, scales)
    assert np.isnan(want).sum() == 96
    assert np.array_equal(np.isnan(k), np.isnan(want))
    big = ~np.isnan(want) & (np.abs(want) >= 2.0 ** -126)  # values that bf16 holds without denormals
    assert np.array_equal(k[big], want[big])
    assert np.all(np.abs(k[~big & ~np.isnan(want)]) <= 2.0 ** -125)


# ---- attention -------------------------------------------------------------------------------
ATTEND = [
    # bits, D, page, Hq, Hkv, (new, length) by sequence, causal, softcap, slopes, max_q, max_kv
    # one token
    (16, 128, 16, 32, 8, [(1, 1)], 1, 0, 0, None, None),
    (16, 128, 16, 32, 8, [(1, 777)], 1, 0, 0, None, None),
    (16, 128, 64, 8, 8, [(1, 31), (1, 33), (1, 0), (0, 50), (1, 128), (1, 129)], 0, 0, 0, None, None),
    (16, 64, 32, 6, 3, [(1, 500), (1, 2)], 1, 30.0, 1, None, None),
    (16, 256, 128, 16, 1, [(1, 300), (1, 65)], 1, 0, 0, None, None),
    (16, 80, 16, 4, 2, [(1, 200)], 1, 0, 1, None, None),
    (16, 32, 256, 4, 4, [(1, 513)], 1, 5.0, 0, None, None),
    (16, 192, 16, 4, 2, [(1, 90)], 1, 0, 0, None, None),
    (4, 128, 32, 32, 8, [(1, 1), (1, 700)], 1, 0, 0, None, None),
    (4, 64, 16, 6, 2, [(1, 47), (1, 48), (1, 0)], 1, 0, 1, None, None),
    (4, 256, 64, 16, 4, [(1, 333)], 1, 50.0, 0, None, None),
    # drafts: one and two row blocks, rows without a key
    (16, 128, 32, 8, 1, [(8, 400), (3, 3), (5, 2)], 1, 0, 1, None, None),
    (16, 64, 16, 8, 2, [(7, 100), (9, 64)], 0, 0, 0, None, None),
    (16, 256, 16, 8, 2, [(8, 70)], 1, 0, 0, None, None),
    (4, 128, 16, 8, 1, [(8, 257), (2, 31)], 1, 20.0, 0, None, None),
    (4, 256, 16, 4, 1, [(9, 90)], 1, 0, 0, None, None),
    (16, 256, 64, 4, 1, [(1, 260), (3, 40)], 1, 12.0, 0, None, None),
    (4, 128, 64, 8, 2, [(4, 700), (1, 20)], 1, 0, 1, None, None),
    (4, 256, 64, 8, 2, [(1, 410), (1, 7)], 1, 0, 0, None, None),
    (16, 256, 32, 8, 2, [(7, 150), (1, 3)], 1, 0, 1, None, None),
    (4, 256, 32, 8, 2, [(8, 90), (5, 5)], 0, 7.0, 0, None, None),
    # two row blocks
    (16, 128, 32, 8, 2, [(7, 400), (3, 2), (5, 129)], 1, 0, 0, None, None),
    (16, 112, 16, 4, 1, [(5, 77), (8, 300)], 1, 11.0, 1, None, None),
    (16, 64, 64, 6, 2, [(10, 200), (1, 31)], 0, 0, 0, None, None),
    (16, 48, 16, 2, 1, [(12, 12), (16, 90)], 1, 0, 1, None, None),
    (4, 128, 128, 8, 2, [(8, 600), (2, 1)], 1, 0, 0, None, None),
    (4, 128, 16, 8, 2, [(6, 99)], 1, 40.0, 0, None, None),
    (4, 64, 32, 4, 1, [(5, 260), (7, 64)], 1, 0, 0, None, None),
    (4, 64, 16, 10, 2, [(6, 65)], 1, 0, 1, None, None),
    # 33 to 64 rows of a kv head: key halves
    (16, 128, 32, 16, 2, [(8, 900), (5, 70), (4, 2)], 1, 0, 1, None, None),
    (16, 128, 16, 8, 1, [(8, 300), (0, 9), (5, 40)], 1, 0, 0, None, None),
    (16, 64, 16, 8, 1, [(8, 300), (0, 9), (6, 6)], 0, 0, 0, None, None),
    (16, 48, 64, 10, 1, [(5, 333), (4, 40)], 1, 9.0, 0, None, None),
    (4, 128, 64, 16, 2, [(7, 500), (8, 33)], 1, 0, 0, None, None),
    (4, 64, 16, 6, 1, [(9, 65), (10, 200)], 1, 30.0, 1, None, None),
    # many sequences, some without rows or keys: the decode line is read 64 sequences at a time
    (16, 64, 16, 4, 2, [(int(i % 7 != 3), i * 37 % 400) for i in range(70)], 1, 0, 0, None, None),
    (4, 64, 16, 2, 1, [(1 + i % 2, i * 53 % 290) for i in range(150)], 1, 0, 0, None, None),
    (16, 32, 16, 2, 2, [(0, 30)] * 65 + [(1, 700), (1, 20)] + [(0, 0)] * 70 + [(2, 300)], 1, 0, 0, None, None),
    (16, 16, 16, 8, 8, [(16, 20)] * 300, 1, 0, 0, 1, None),       # more rows than partial slots
    # prompts
    (16, 128, 64, 4, 2, [(130, 130), (40, 100), (1, 5)], 1, 0, 0, None, None),
    (16, 128, 16, 8, 1, [(33, 20), (17, 300)], 1, 0, 0, None, None),
    (16, 64, 32, 3, 3, [(200, 333)], 0, 15.0, 1, None, None),
    (16, 96, 128, 2, 1, [(300, 300)], 1, 0, 0, None, None),
    (16, 256, 32, 4, 2, [(70, 140)], 1, 0, 1, None, None),
    (16, 16, 16, 5, 5, [(129, 129)], 1, 0, 0, None, None),
    (4, 128, 16, 8, 2, [(65, 130), (100, 100)], 1, 0, 0, None, None),
    (4, 64, 64, 6, 2, [(150, 400)], 1, 50.0, 1, None, None),
    (4, 256, 32, 4, 1, [(40, 77)], 0, 0, 0, None, None),
    (16, 256, 16, 2, 2, [(66, 200), (90, 90)], 1, 0, 0, None, None),
    (4, 256, 64, 2, 1, [(50, 120)], 1, 6.0, 0, None, None),
    (4, 64, 16, 4, 1, [(50, 60)], 1, 0, 0, None, None),
    (4, 128, 16, 4, 1, [(50, 260)], 0, 0, 1, None, None),
    (16, 128, 32, 4, 1, [(50, 260)], 1, 6.0, 0, None, None),
    (4, 64, 32, 16, 1, [(4, 100)], 1, 0, 0, None, None),
    # more row tiles than CUs
    *[(bits, D, 16, 8, 8, [(70 + i % 60, 3 * i + 20) for i in range(40)], 0, cap, 0, None, None)
      for bits, D in ((16, 128), (16, 64), (4, 128), (4, 64)) for cap in (0, 25.0)],
    # four parts of a row, and many
    (4, 64, 32, 16, 2, [(8, 100 + 10 * i) for i in range(31)] + [(5, 512)], 1, 0, 0, None, None),
    (16, 128, 64, 8, 2, [(1, 5000), (1, 2500)], 1, 0, 0, None, None),
    # bounds that sequences pass: rows and keys behind them are served too
    (16, 128, 16, 8, 2, [(9, 300), (50, 60)], 1, 0, 0, 1, 16),
    (16, 128, 64, 8, 8, [(300, 700)], 1, 0, 0, 70, 200),
    (4, 128, 32, 4, 1, [(20, 999), (1, 400)], 1, 0, 0, 1, 130),
    # and bounds far above them: parts without a key
    (16, 128, 16, 8, 2, [(2, 30), (1, 200)], 1, 0, 0, 4, 20000),
    (4, 64, 16, 8, 2, [(70, 100), (3, 700)], 1, 0, 0, 100, 9000),
]


@pytest.mark.parametrize("case", ATTEND, ids=["%d-%d-%d-%d-%d-%s" % (*c[:5], "_".join(map(str, c[5][0])))
                                              for c in ATTEND])
def test_attend(case):
    bits, D, page, Hq, Hkv, seqs, causal, softcap, slopes, max_q, max_kv = case
    print("attend", case, flush=True)
    c = pu.Cache(seqs, Hkv, D, page, bits, 3)
    c.fill(31)
    q = pu.normal((c.N, Hq, D), 5, 2.0)
    sl = np.exp2(-8.0 * np.arange(1, Hq + 1) / Hq).astype(np.float32) if slopes else None
    ref, bound = pu.attend_ref(c, q, Hq, causal, 0.0, softcap, sl)
    O = pu.attend(c, q, Hq, causal, 0.0, softcap, sl, max_q, max_kv, stride=64)
    check(O, ref, bound, case)
    again = pu.attend(c, q, Hq, causal, 0.0, softcap, sl, max_q, max_kv, stride=64)
    assert np.array_equal(O, again)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n", [1, 6, 80])
def test_attend_hides_pages_that_are_none(bits, n):
    """Entries outside the cache, in the middle and at the end of a tile, and a whole row of them."""
    D, Hkv, Hq, page = 128, 2, 8, 16
    c = pu.Cache([(n, 300), (n, 100), (n, 90)], Hkv, D, page, bits, 3)
    c.fill(13)
    q = pu.normal((c.N, Hq, D), 5)
    hidden = [(0, 0), (0, 5), (0, 18), (1, 6)] + [(2, i) for i in range(6)]
    keep = c.table.copy()
    for i, (b, col) in enumerate(hidden):
        c.table[b, col] = (-1, c.pages, 2 ** 31 - 1, -2 ** 31)[i % 4]
    desc = c.device()
    c.table = keep  # the reference reads the rows and hides them
    ref, bound = pu.attend_ref(c, q, Hq, 1, hidden=hidden)
    O = pu.attend(c, q, Hq, 1, desc=desc)
    check(O, ref, bound, (bits, n))
    assert np.all(O[c.start[2]:] == 0)


@pytest.mark.parametrize("n", [1, 40])
def test_attend_lengths_and_starts_of_any_kind(n):
    """Lengths past the table's row are cut, negative ones are none; starts stay in the token tensors."""
    D, Hkv, Hq, page = 64, 1, 4, 32
    c = pu.Cache([(n, 200), (n, 64)], Hkv, D, page, 16, 3, cols=2)
    c.fill(7)
    q = pu.normal((c.N, Hq, D), 5)
    ref, bound = pu.attend_ref(c, q, Hq, 0)
    check(pu.attend(c, q, Hq, 0), ref, bound, n)
    c.kv_len = np.array([-2 ** 31, 64], np.int32)
    O = pu.attend(c, q, Hq, 1, max_kv=64)
    assert np.all(O[:n] == 0) and np.any(O[n:] != 0)
    # two sequences, the second's end past the tensors
    full = c.start.copy()
    c.start = np.array([0, n, 2 ** 31 - 1], np.int32)
    c.kv_len = np.array([64, 64], np.int32)
    T = 2 * n
    with ts.DeviceBuffer.from_array(q) as dq, ts.DeviceBuffer(q.nbytes) as do, \
            ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds:
        do.fill_bytes(0xFF)
        ts.attn_paged(c.device(), ts.Rows(dq, Hq * D, D), ts.Rows(do, Hq * D, D), T, Hq, 0, None, n, 64, ds)
        ts.synchronize()
        assert np.all(np.isfinite(pu.f32(do.download(np.uint16))))
        for start in ([-5, n, 2 * n], [2 ** 31 - 1, -3, 0], [n, 0, n]):
            c.start = np.array(start, np.int32)
            ts.attn_paged(c.device(), ts.Rows(dq, Hq * D, D), ts.Rows(do, Hq * D, D), T, Hq, 0, None, n, 64,
                          ds)
            ts.synchronize()
    c.start = full


def test_split_parts_join():
    """One sequence's keys over many workgroups, parts of which a row's causal limit leaves empty."""
    for bits, Hq, Hkv, n, kv in ((16, 8, 2, 1, 5000), (4, 4, 1, 3, 4097), (16, 4, 1, 60, 2000),
                                 (16, 2, 2, 300, 1000)):
        print("split", bits, n, kv, flush=True)
        c = pu.Cache([(n, kv), (n, 100)], Hkv, 128, 64, bits, 3)
        c.fill(17)
        plan = ts.attn_paged_plan(c.device(), c.N, Hq, 1, None, n, kv)
        assert plan[-1][0].startswith("attn_paged_merge_kernel<"), plan
        q = pu.normal((c.N, Hq, 128), 5, 3.0)
        ref, bound = pu.attend_ref(c, q, Hq, 1)
        check(pu.attend(c, q, Hq, 1), ref, bound, (bits, n, kv))


@pytest.mark.parametrize("bits,n", [(16, 1), (16, 70), (4, 1), (4, 70)])
def test_scores_far_apart(bits, n):
    """Scores that rise by hundreds from tile to tile, and fall again: the running maximum follows."""
    D, page = 64, 32
    c = pu.Cache([(n, 500)], 1, D, page, bits, 3)
    K, V = pu.normal((500, 1, D), 1), pu.normal((500, 1, D), 2)
    ramp = np.concatenate([np.linspace(0.1, 60, 300), np.linspace(60, 0.1, 200)]).astype(np.float32)
    K = pu.bf16(pu.f32(K) * ramp[:, None, None])
    c.put(0, 0, K, V)
    q = pu.normal((n, 2, D), 5, 4.0)
    ref, bound = pu.attend_ref(c, q, 2, 1)
    check(pu.attend(c, q, 2, 1), ref, bound, (bits, n))


@pytest.mark.parametrize("bits,n,kv", [(16, 1, 100), (16, 1, 5000), (4, 1, 5000), (16, 8, 4000), (4, 20, 3000),
                                       (16, 100, 2000), (4, 100, 700), (16, 40, 64)])
def test_nan_and_infinities_stay_in_their_rows(bits, n, kv):
    """A NaN or an infinity in a row of q, or a NaN in a key, makes NaN of the rows that meet it, whole or in
    parts, and of no other."""
    Hq, Hkv, D = 4, 2, 128
    c = pu.Cache([(n, kv), (n, kv // 2)], Hkv, D, 32, bits, 3)
    c.fill(23)
    pg, at = c.places(0, kv - (n + 1) // 2, kv)  # the key of a row in the middle of the new ones
    x, nan = (c.ks, 255) if bits == 4 else (c.k, 0xFF)
    x[pg[0], 1, at[0]] = nan
    q = pu.normal((c.N, Hq, D), 5)
    ref, bound = pu.attend_ref(c, q, Hq, 1)
    lost = np.isnan(ref).any(-1)
    assert lost.sum() == 2 * ((n + 1) // 2)
    q[0, 0, 5] = 0x7FC0  # NaN
    q[c.N - 1, 0, 7] = 0x7F80  # inf
    lost[0, 0] = lost[c.N - 1, 0] = True
    o = pu.attend(c, q, Hq, 1, poison=0x3F)
    print(np.isnan(o).all(-1).sum(), lost.sum())
    assert np.array_equal(np.isnan(o).any(-1), lost) and np.array_equal(np.isnan(o).all(-1), lost)
    check(np.where(lost[..., None], 0, o), np.where(lost[..., None], 0, ref),
          np.where(lost[..., None], 0, bound), (bits, n, kv))


def test_cache_past_4_gib():
    """Pages whose byte offsets pass 32 bits."""
    D, Hkv, page = 128, 8, 256
    per = Hkv * page * D * 2
    pages = (5 << 30) // per
    ids = np.array([pages - 1, 3, pages - 2, (2 << 30) // per, (4 << 30) // per], np.int32)
    kv = 256 * 4 + 90
    K, V = pu.normal((kv, Hkv, D), 1), pu.normal((kv, Hkv, D), 2)
    for n, Hq in ((1, 16), (20, 32)):
        c = pu.Cache([(n, kv)], Hkv, D, page, 16, 1)
        c.put(0, 0, K, V)
        with ts.DeviceBuffer(pages * per) as dk, ts.DeviceBuffer(pages * per) as dv:
            for i, pg in enumerate(ids):
                pu.memcpy_to(dk.ptr + int(pg) * per, c.k[c.table[0, i]])
                pu.memcpy_to(dv.ptr + int(pg) * per, c.v[c.table[0, i]])
            base = c.device()
            table = c.table.copy()
            table[0, :5] = ids
            with ts.DeviceBuffer.from_array(table) as dt:
                desc = ts.KvCache(dk, dv, dt, base.kv_len, base.q_start, 1, c.cols, pages, page, Hkv, D)
                q = pu.normal((n, Hq, D), 5)
                ref, bound = pu.attend_ref(c, q, Hq, 1)
                check(pu.attend(c, q, Hq, 1, desc=desc), ref, bound, n)
                with ts.DeviceBuffer(kv * Hkv * D * 2) as ok, ts.DeviceBuffer(kv * Hkv * D * 2) as ov, \
                        ts.DeviceBuffer.from_array(np.array([0, kv], np.int32)) as st:
                    desc.q_start = st.ptr
                    ts.attn_kv_read(desc, ts.Rows(ok, Hkv * D, D), ts.Rows(ov, Hkv * D, D), kv, kv)
                    ts.synchronize()
                    assert np.array_equal(ok.download(np.uint16).reshape(K.shape), K)
                    assert np.array_equal(ov.download(np.uint16).reshape(V.shape), V)


# ---- together --------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 4])
def test_generation(bits):
    """Two prompts of unequal length, then tokens one by one: append and attend as a server does, every step
    against the tokens so far."""
    D, Hq, Hkv, page = 128, 8, 2, 16
    rope = pu.rope_table(200, D)
    lens = [0, 0]
    c = pu.Cache([(1, 140), (1, 60)], Hkv, D, page, bits, 3)
    for step, new in enumerate([(90, 37), (30, 1), (1, 1), (1, 1), (0, 1), (1, 1)]):
        lens = [a + n for a, n in zip(lens, new)]
        c.seqs = list(zip(new, lens))
        c.start = np.array([0, new[0], sum(new)], np.int32)
        c.kv_len, c.N = np.array(lens, np.int32), sum(new)
        qkv = pu.normal((c.N, Hq + 2 * Hkv, D), 100 + step)
        q = append(c, qkv, Hq, rope, D, 0)
        for b, n in enumerate(new):
            r = slice(c.start[b], c.start[b + 1])
            pos = np.arange(lens[b] - n, lens[b])
            assert np.array_equal(q[r], pu.rotate(qkv[r, :Hq], pos, rope, D, 0))
        ref, bound = pu.attend_ref(c, q, Hq, 1)
        check(pu.attend(c, q, Hq, 1), ref, bound, step)


@pytest.mark.parametrize("bits", [16, 4])
def test_read_back_gives_attn_flash_the_same_attention(bits):
    """attn_kv_read into the dense layout, attn_flash on it, attn_paged on the cache."""
    D, Hq, Hkv, n, kv = 128, 8, 2, 100, 250
    c = pu.Cache([(n, kv)], Hkv, D, 32, bits, 3)
    c.fill(5)
    q = pu.normal((n, Hq, D), 9)
    ref, bound = pu.attend_ref(c, q, Hq, 1)
    O = pu.attend(c, q, Hq, 1)
    check(O, ref, bound, bits)
    c.start = np.array([0, kv], np.int32)
    with ts.DeviceBuffer(kv * Hkv * D * 2) as dk, ts.DeviceBuffer(kv * Hkv * D * 2) as dv, \
            ts.DeviceBuffer.from_array(np.ascontiguousarray(q.transpose(1, 0, 2))) as dq, \
            ts.DeviceBuffer(n * Hq * D * 4) as do, \
            ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds:
        ts.attn_kv_read(c.device(), ts.Rows(dk, D, kv * D), ts.Rows(dv, D, kv * D), kv, kv)
        ts.attn_flash(dq, dk, dv, do, Hq, Hkv, n, kv, D, 1, 128, ds)
        ts.synchronize()
        dense = do.download(np.float32).reshape(Hq, n, D).transpose(1, 0, 2)
    check(dense, ref, bound, bits)


def test_graph_replays_with_other_lengths():
    """One captured step (append, attend, the join of the parts) replayed with new tokens, lengths and pages,
    each time against the same step run eagerly."""
    D, Hq, Hkv, page, B, cols = 128, 8, 2, 16, 3, 40
    hip = pu.Hip()
    c = pu.Cache([(1, cols * page)] * B, Hkv, D, page, 16, 3, spare=0, cols=cols)
    c.fill(5)
    c.device()
    clean = {n: getattr(c, n).copy() for n in ("k", "v")}
    rope = pu.rope_table(cols * page, D)
    H = Hq + 2 * Hkv
    with ts.DeviceBuffer(B * H * D * 2) as dx, ts.DeviceBuffer(B * Hq * D * 2) as dq, \
            ts.DeviceBuffer(B * Hq * D * 2) as do, ts.DeviceBuffer.from_array(rope) as dr, \
            ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds:
        desc = c.device()
        assert len(ts.attn_paged_plan(desc, B, Hq, 1, None, 1, cols * page)) == 2

        def step():
            ts.attn_kv_append(desc, ts.Rows(dx, H * D, D), ts.Rows(dq, Hq * D, D),
                              ts.Rows(dx.ptr + 2 * Hq * D, H * D, D),
                              ts.Rows(dx.ptr + 2 * (Hq + Hkv) * D, H * D, D), B, Hq, dr, len(rope), D)
            ts.attn_paged(desc, ts.Rows(dq, Hq * D, D), ts.Rows(do, Hq * D, D), B, Hq, 1, None, 1,
                          cols * page, ds)

        st = hip.stream()
        ex = hip.capture(st, step)
        lens = np.array([0, 300, 17], np.int32)
        for it in range(5):
            lens = lens + 1 + 100 * (it == 3)
            c.kv_len = lens.astype(np.int32)
            c.table = np.random.default_rng(it).permutation(c.pages)[:B * cols].astype(np.int32)
            c.table = c.table.reshape(B, cols)
            got = []
            for run in (lambda: hip("hipGraphLaunch", ex, st), step):
                c.k, c.v = clean["k"].copy(), clean["v"].copy()
                c.device()
                dx.upload(pu.normal((B, H, D), 40 + it))
                do.fill_bytes(0xFF)
                ts.synchronize()
                run()
                ts.synchronize()
                c.download()
                got.append((do.download(np.uint16), c.k.copy(), c.v.copy()))
            for a, b in zip(*got):
                assert np.array_equal(a, b), it
            O = pu.f32(got[0][0]).reshape(B, Hq, D)
            c.seqs, c.start, c.N = [(1, int(n)) for n in lens], np.arange(B + 1, dtype=np.int32), B
            ref, bound = pu.attend_ref(c, dq.download(np.uint16).reshape(B, Hq, D), Hq, 1)
            check(O, ref, bound, it)
            c.seqs = [(1, cols * page)] * B


def test_two_streams_at_once():
    """Two calls with a scratch each, on streams of their own, against the same calls one by one."""
    D, Hq, Hkv, kv = 128, 8, 2, 3000
    hip = pu.Hip()
    cs = [pu.Cache([(1, kv), (1, 500)], Hkv, D, 64, 16, s) for s in (1, 2)]
    calls = []
    for i, c in enumerate(cs):
        c.fill(50 + 10 * i)
        calls.append((c.device(), ts.DeviceBuffer.from_array(pu.normal((2, Hq, D), 7 + i)),
                      ts.DeviceBuffer(2 * Hq * D * 2), ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128))))

    def go(i):
        desc, q, o, s = calls[i]
        ts.attn_paged(desc, ts.Rows(q, Hq * D, D), ts.Rows(o, Hq * D, D), 2, Hq, 1, None, 1, kv, s)

    go(0), go(1)
    ts.synchronize()
    alone = [c[2].download(np.uint16) for c in calls]
    for c in calls:
        c[2].fill_bytes(0xFF)
    ts.synchronize()
    streams = [hip.stream() for _ in calls]
    try:
        for _ in range(20):
            for i, s in enumerate(streams):
                ts.set_stream(s.value)
                go(i)
    finally:
        ts.set_stream(None)
    ts.synchronize()
    for a, c in zip(alone, calls):
        assert np.array_equal(a, c[2].download(np.uint16))
