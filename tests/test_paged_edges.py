"""The paged KV cache on the GPU where a mistake could hide from the other tests: a caller's own scale, other orders of
q, k, v and o, starts of any kind with guards around the rows, keys at the edges of tiles, pages and parts that carry a
row each, and token tensors far larger than the sequences' rows."""
import numpy as np
import pytest

import paged_util as pu
import transfer_station_amd as ts
from test_paged import check
from transfer_station_amd import _lib


def memcpy_from(ptr, shape):
    out = np.empty(shape, np.uint16)
    _lib.check(_lib.lib().attn_dev_memcpy_dtoh(out.ctypes.data, ptr, out.nbytes), "hipMemcpy")
    return out


# One of each kernel: bits, D, page, Hq, Hkv, (new, length) by sequence.
KERNELS = [
    (16, 64, 16, 8, 2, [(1, 700), (1, 33)]),
    (16, 128, 64, 8, 1, [(2, 600), (1, 90)]),
    (16, 256, 32, 8, 2, [(1, 300), (3, 40)]),
    (4, 64, 16, 4, 2, [(1, 500)]),
    (4, 256, 64, 8, 2, [(1, 410)]),
    (16, 128, 32, 8, 2, [(7, 300), (1, 12)]),
    (4, 64, 32, 4, 1, [(5, 260)]),
    (16, 128, 16, 8, 1, [(8, 500), (3, 7)]),
    (16, 128, 32, 64, 1, [(1, 400), (1, 20)]),  # 64 rows of one token
    (4, 128, 64, 16, 2, [(7, 300)]),
    (16, 64, 32, 6, 3, [(70, 333), (1, 90)]),
    (4, 128, 16, 4, 1, [(50, 260)]),
    (16, 256, 32, 4, 2, [(70, 140)]),
    (4, 256, 32, 4, 1, [(80, 130)]),
]
IDS = ["%d-%d-%d" % (c[0], c[1], i) for i, c in enumerate(KERNELS)]


@pytest.mark.gpu
@pytest.mark.parametrize("scale,cap,slopes", [(0.01, 0, 0), (0.9, 0, 0), (0.9, 20.0, 0), (0.3, 0, 1)])
@pytest.mark.parametrize("case", KERNELS, ids=IDS)
def test_own_scale(case, scale, cap, slopes):
    bits, D, page, Hq, Hkv, seqs = case
    print("scale", case, scale, cap, slopes, flush=True)
    c = pu.Cache(seqs, Hkv, D, page, bits, 3)
    c.fill(31)
    q = pu.normal((c.N, Hq, D), 5)
    sl = np.exp2(-8.0 * np.arange(1, Hq + 1) / Hq).astype(np.float32) if slopes else None
    ref, bound = pu.attend_ref(c, q, Hq, 1, scale, cap, sl)
    check(pu.attend(c, q, Hq, 1, scale, cap, sl), ref, bound, (case, scale, cap, slopes))


@pytest.mark.gpu
@pytest.mark.parametrize("case", KERNELS, ids=IDS)
def test_heads_outside_tokens(case):
    """q as [heads][tokens][D] and o as [tokens][heads][D] with gaps, then the other way round."""
    bits, D, page, Hq, Hkv, seqs = case
    print("heads", case, flush=True)
    c = pu.Cache(seqs, Hkv, D, page, bits, 3)
    c.fill(31)
    q = pu.normal((c.N, Hq, D), 5)
    ref, bound = pu.attend_ref(c, q, Hq, 1)
    T, gap = c.N + 2, 24
    for turned in (0, 1):
        # (token, head) strides of q and o, and their tensors' sizes
        major, minor = (D, (T + 1) * D), (Hq * (D + gap) + 8, D + gap)
        (qt, qh), (ot, oh) = (major, minor) if turned == 0 else (minor, major)
        qbuf = np.full(max(T * qt, Hq * qh) + D, 0xFFFF, np.uint16)
        at = np.arange(c.N)[:, None, None] * qt + np.arange(Hq)[:, None] * qh + np.arange(D)
        qbuf[at] = q
        osize = max(T * ot, Hq * oh) + D
        with ts.DeviceBuffer.from_array(qbuf) as dq, ts.DeviceBuffer(osize * 2) as do, \
                ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds:
            do.fill_bytes(0xFF)
            ts.attn_paged(c.device(), ts.Rows(dq, qt, qh), ts.Rows(do, ot, oh), T, Hq, 1, None,
                          max(n for n, _ in seqs), max(k for _, k in seqs), ds)
            ts.synchronize()
            raw = do.download(np.uint16)
        at = np.arange(c.N)[:, None, None] * ot + np.arange(Hq)[:, None] * oh + np.arange(D)
        check(pu.f32(raw[at]), ref, bound, (case, turned))
        raw[at] = 0xFFFF
        assert np.all(raw == 0xFFFF)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,D,Hq,Hkv,rot,pairs", [(16, 128, 8, 2, 128, 0), (16, 80, 3, 3, 32, 1), (4, 64, 6, 2, 64, 0),
                                                     (4, 256, 2, 1, 128, 1)])
def test_append_and_read_heads_outside_tokens(bits, D, Hq, Hkv, rot, pairs):
    """q, q_out, k and v, and the rows read back, as [heads][tokens][D], each with a stride of its own."""
    seqs = [(9, 30), (1, 17), (4, 4)]
    want, got = (pu.Cache(seqs, Hkv, D, 16, bits, 5) for _ in range(2))
    N, T = got.N, got.N + 2
    rope = pu.rope_table(40, rot)
    q, k, v = (pu.normal((h, T + i, D), 70 + i) for i, h in enumerate((Hq, Hkv, Hkv)))
    with ts.DeviceBuffer.from_array(q) as dq, ts.DeviceBuffer.from_array(k) as dk, \
            ts.DeviceBuffer.from_array(v) as dv, ts.DeviceBuffer(Hq * (T + 3) * D * 2) as dqo, \
            ts.DeviceBuffer.from_array(rope) as dr, ts.DeviceBuffer(Hkv * (T + 4) * D * 2) as bk, \
            ts.DeviceBuffer(Hkv * (T + 5) * D * 2) as bv:
        for d in (dqo, bk, bv):
            d.fill_bytes(0xFF)
        ts.attn_kv_append(got.device(), ts.Rows(dq, D, T * D), ts.Rows(dqo, D, (T + 3) * D),
                          ts.Rows(dk, D, (T + 1) * D), ts.Rows(dv, D, (T + 2) * D), T, Hq, dr, len(rope), rot,
                          pairs, 9)
        ts.synchronize()
        got.download()
        ts.attn_kv_read(got.device(), ts.Rows(bk, D, (T + 4) * D), ts.Rows(bv, D, (T + 5) * D), T, 9)
        ts.synchronize()
        qo = dqo.download(np.uint16).reshape(Hq, T + 3, D)
        back = [bk.download(np.uint16).reshape(Hkv, T + 4, D), bv.download(np.uint16).reshape(Hkv, T + 5, D)]
    q, k, v = (x.transpose(1, 0, 2) for x in (q, k, v))
    for b, (n, kv) in enumerate(seqs):
        r, pos = slice(want.start[b], want.start[b + 1]), np.arange(kv - n, kv)
        assert np.array_equal(qo[:, r].transpose(1, 0, 2), pu.rotate(q[r], pos, rope, rot, pairs))
        want.put(b, kv - n, pu.rotate(k[r], pos, rope, rot, pairs), v[r])
    for x in ("k", "v") + (("ks", "vs") if bits == 4 else ()):
        assert np.array_equal(getattr(got, x), getattr(want, x)), x
    assert np.all(qo[:, N:] == 0xFFFF)
    for i, x in enumerate(back):
        assert np.all(x[:, N:] == 0xFFFF)
        for b, (n, kv) in enumerate(seqs):
            rows = pu.f32(x[:, want.start[b]:want.start[b + 1]]).astype(np.float64)
            assert np.array_equal(rows.transpose(1, 0, 2), want.get(b, kv - n, kv)[i])


STARTS = [
    # starts, the rows that are some sequence's: (sequence, first row, rows), with n rows each meant
    (lambda n, T: [-5, n, 2 * n], lambda n, T: [(0, 0, n), (1, n, n)]),
    (lambda n, T: [0, n, 2 ** 31 - 1], lambda n, T: [(0, 0, n), (1, n, T - n)]),
    (lambda n, T: [2 ** 31 - 1, -3, 0], lambda n, T: []),
    (lambda n, T: [-2 ** 31, -1, -1], lambda n, T: []),
    (lambda n, T: [n, 0, n], lambda n, T: [(1, 0, n)]),
    (lambda n, T: [T, T, T], lambda n, T: []),
    (lambda n, T: [T - 1, T + 5, T + 9], lambda n, T: [(0, T - 1, 1)]),
    (lambda n, T: [n, 2 * n, n], lambda n, T: [(0, n, n)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n", [1, 5, 12, 40])
@pytest.mark.parametrize("which", range(len(STARTS)))
def test_starts_of_any_kind(bits, n, which):
    """Starts that fall, are negative or lie past the tensors: the rows that they name are right, all others and the
    memory around them stay as they were. With 4 query heads on one kv head, n tokens are 4, 20, 48 or 160 rows."""
    D, Hkv, Hq, page, kv, guard = 64, 1, 4, 32, 64, 64
    print("starts", bits, n, which, flush=True)
    T = 2 * n + 1
    start, rows = STARTS[which][0](n, T), STARTS[which][1](n, T)
    full = pu.Cache([(n, kv), (n, kv)], Hkv, D, page, bits, 3)
    full.fill(7)
    full.start = np.array(start, np.int32)
    x = pu.normal((T, Hq + 2 * Hkv, D), 5)
    W = (Hq + 2 * Hkv) * D
    buf = np.full((T + 2 * guard, W), 0xFFFF, np.uint16)
    buf[guard:guard + T] = x.reshape(T, W)
    rope = pu.rope_table(kv, D)
    out = {}
    with ts.DeviceBuffer.from_array(buf) as dx, ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds, \
            ts.DeviceBuffer.from_array(rope) as dr:
        p = dx.ptr + guard * W * 2
        q, k, v = (ts.Rows(p + 2 * D * h, W, D) for h in (0, Hq, Hq + Hkv))
        outs = {y: ts.DeviceBuffer(buf.nbytes) for y in ("o", "q", "kv")}
        at = {y: d.ptr + guard * W * 2 for y, d in outs.items()}
        for d in outs.values():
            d.fill_bytes(0xFF)
        desc = full.device()
        ts.attn_paged(desc, q, ts.Rows(at["o"], W, D), T, Hq, 0, None, n, kv, ds)
        ts.attn_kv_read(desc, ts.Rows(at["kv"], W, D), ts.Rows(at["kv"] + 2 * D, W, D), T, n)
        ts.synchronize()
        ref = pu.Cache([(m, kv) for _, _, m in rows], Hkv, D, page, bits, 3)
        ref.table = full.table[[b for b, _, _ in rows]] if rows else ref.table
        ref.pages, ref.k, ref.v, ref.ks, ref.vs = full.pages, full.k, full.v, full.ks, full.vs
        before = {y: getattr(full, y).copy() for y in ("k", "v", "ks", "vs")}
        qs = np.concatenate([x[r0:r0 + m, :Hq] for _, r0, m in rows] or [x[:0, :Hq]])
        O, bound = pu.attend_ref(ref, qs, Hq, 0) if rows else (None, None)
        back = [ref.get(i, kv - m, kv) for i, (_, _, m) in enumerate(rows)]
        ts.attn_kv_append(desc, q, ts.Rows(at["q"], W, D), k, v, T, Hq, dr, kv, D, 0, n)
        ts.synchronize()
        full.download()
        for y, d in outs.items():
            out[y] = d.download(np.uint16).reshape(buf.shape)
            d.free()
    mine = np.zeros(T + 2 * guard, bool)
    for i, (b, r0, m) in enumerate(rows):
        r = slice(guard + r0, guard + r0 + m)
        mine[r] = True
        pos = np.arange(kv - m, kv)
        lo = ref.start[i]
        check(pu.f32(out["o"][r, :Hq * D]).reshape(m, Hq, D), O[lo:lo + m], bound[lo:lo + m], (bits, n, which))
        assert np.array_equal(out["q"][r, :Hq * D].reshape(m, Hq, D),
                              pu.rotate(x[r0:r0 + m, :Hq], pos, rope, D, 0))
        for j in (0, 1):
            got = pu.f32(out["kv"][r, j * D:(j + 1) * D]).astype(np.float64)
            assert np.array_equal(got, back[i][j][:, 0])
        want = pu.Cache([(m, kv)], Hkv, D, page, bits, 3)
        want.table, want.pages = full.table[b:b + 1], full.pages
        want.k, want.v, want.ks, want.vs = before["k"], before["v"], before["ks"], before["vs"]
        want.put(0, kv - m, pu.rotate(x[r0:r0 + m, Hq:Hq + Hkv], pos, rope, D, 0), x[r0:r0 + m, Hq + Hkv:])
    for y in before:  # the pages of the rows' sequences as appended to, the others as they were
        assert np.array_equal(getattr(full, y), before[y]), y
    for y in out:
        assert np.all(out[y][~mine] == 0xFFFF), y
        assert np.all(out[y][:, (2 * Hkv if y == "kv" else Hq) * D:] == 0xFFFF), y


def planted(bits, D, Hkv, g, page, kv, n, seed=3):
    """A cache of one sequence, and rows of q that each look at one pair of keys: (cache, q [n][Hq][D], pairs). The
    pairs are keys at the edges of 16, 32, 128, the page and everything that 128 divides, each beside a key elsewhere
    with the same K row, so that a row's output is the mean of two V rows: a key that is left out leaves the other,
    and one that is taken twice weighs two to one."""
    rng = np.random.default_rng(seed)
    c = pu.Cache([(n, kv)], Hkv, D, page, bits, seed)
    K, V = pu.normal((kv, Hkv, D), 1), pu.normal((kv, Hkv, D), 2)
    old = kv - n  # every row sees these
    edges = sorted({e for s in (16, 32, page) for e in (0, s - 1, s, old // s * s - 1)} |
                   {e for m in range(128, old, 128) for e in (m - 1, m)} | {old - 1})
    edges = [e for e in edges if 0 <= e < old]
    free = np.array([j for j in range(old) if j not in set(edges)])
    other = rng.choice(free, len(edges), replace=False)
    K[other] = K[edges]
    c.put(0, 0, K, V)
    held = c.get(0, 0, kv)[0]
    rows = [(i, h) for i in range(n) for h in range(Hkv * g)]
    picks = [(edges[m], int(other[m])) for m in range(len(edges))]
    calls = []
    for lo in range(0, len(picks), len(rows)):
        q, pairs = np.zeros((n, Hkv * g, D), np.float32), {}
        for (i, h), pr in zip(rows, picks[lo:lo + len(rows)]):
            x = held[pr[0], h // g]
            q[i, h] = x * (40.0 * D ** 0.5 / (x @ x))  # a score of 40, and of 40 / sqrt(D) times a normal elsewhere
            pairs[i, h] = pr
        calls.append((pu.bf16(q), pairs))
    return c, calls


PLANTED = [
    # bits, D, Hkv, heads per kv head, page, kv, n, further sequences beside it
    (16, 128, 2, 4, 64, 5000, 1, []),
    (16, 128, 2, 4, 64, 5000, 1, [(1, 2500), (1, 130), (0, 70), (1, 0), (1, 700)]),
    (16, 256, 1, 8, 16, 3001, 1, [(1, 400)]),
    (4, 64, 2, 4, 32, 4097, 1, [(1, 1000)]),
    (4, 128, 1, 8, 128, 2900, 1, []),
    (4, 256, 1, 8, 64, 2050, 2, []),
    (16, 64, 1, 4, 16, 2000, 8, [(3, 900)]),
    (4, 128, 1, 4, 32, 1999, 7, [(8, 77)]),
    (16, 128, 1, 8, 32, 3000, 8, [(5, 200)]),
    (4, 64, 1, 8, 16, 2100, 7, []),
    (16, 128, 2, 4, 64, 4100, 60, []),
    (16, 64, 1, 4, 128, 1500, 70, [(9, 60)]),
    (4, 128, 1, 4, 16, 1600, 50, []),
    (16, 256, 1, 2, 32, 1300, 90, []),
    (4, 256, 1, 2, 64, 1200, 66, []),
]


def with_others(c, others):
    """The same cache with further sequences behind the first."""
    if not others:
        return c
    seqs = c.seqs + others
    w = pu.Cache(seqs, c.Hkv, c.D, c.page, c.bits, 8)
    w.fill(900)
    (n, kv), (pg, at), (pg2, at2) = c.seqs[0], c.places(0, 0, c.seqs[0][1]), w.places(0, 0, c.seqs[0][1])
    for x in ("k", "v", "ks", "vs"):
        getattr(w, x)[pg2, :, at2] = getattr(c, x)[pg, :, at]
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [1, 0])
@pytest.mark.parametrize("case", PLANTED, ids=["%d-%d-%d" % (c[0], c[1], i) for i, c in enumerate(PLANTED)])
def test_every_key_at_an_edge_counts_once(case, causal):
    bits, D, Hkv, g, page, kv, n, others = case
    print("planted", case, causal, flush=True)
    c, calls = planted(bits, D, Hkv, g, page, kv, n)
    w = with_others(c, others)
    for q, pairs in calls:
        x = np.concatenate([q, pu.normal((w.N - n, Hkv * g, D), 9)])
        O = pu.attend(w, x, Hkv * g, causal)
        ref, bound = pu.attend_ref(c, q, Hkv * g, causal)
        for i, h in pairs:
            off = np.abs(O[i, h] - ref[i, h]) - bound[i, h]
            assert off.max() <= 0, (case, pairs[i, h], float(off.max()))


def test_the_planted_keys_show_a_mistake():
    """The oracle with a key left out, or taken twice, is further off than the bound in every planted row."""
    for bits, D, Hkv, g, page, kv, n, _ in PLANTED[::3]:
        c, calls = planted(bits, D, Hkv, g, page, kv, n)
        K, V = c.get(0, 0, kv)
        for q, pairs in calls[:2]:
            ref, bound = pu.attend_ref(c, q, Hkv * g, 0)
            for (i, h), (j, k) in pairs.items():
                s = D ** -0.5 * (K[:, h // g] @ pu.f32(q[i, h]).astype(np.float64))
                w = np.exp(s - s.max())
                assert np.all(np.abs((w / w.sum()) @ V[:, h // g] - ref[i, h]) <= 1e-9)
                for f in (0.0, 2.0):
                    for key in (j, k):
                        x = w.copy()
                        x[key] *= f
                        off = np.abs((x / x.sum()) @ V[:, h // g] - ref[i, h]) - bound[i, h]
                        assert off.max() > 0.1, (bits, D, j, k)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("pad", [0, 500, 2000, 20000])
def test_token_tensors_far_larger_than_the_rows(bits, pad):
    """T bounds the rows, and with it the parts that the scratch holds: fewer of them, then none, the same results
    within the bound."""
    D, Hq, Hkv = 64, 32, 4
    c = pu.Cache([(1, 3000), (1, 200), (0, 90), (1, 1)], Hkv, D, 32, bits, 3)
    c.fill(11)
    q = pu.normal((c.N, Hq, D), 5)
    ref, bound = pu.attend_ref(c, q, Hq, 1)
    check(pu.attend(c, q, Hq, 1, pad=pad), ref, bound, (bits, pad))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_single_tokens_beside_a_chunk(bits, D):
    """A step of a server: one chunk of a long prompt, drafts, and single tokens of all lengths."""
    Hq, Hkv = 8, 2
    c = pu.Cache([(1, 900), (150, 700), (1, 1), (8, 333), (1, 64), (0, 200), (1, 1500)], Hkv, D, 16, bits, 3)
    c.fill(11)
    q = pu.normal((c.N, Hq, D), 5)
    ref, bound = pu.attend_ref(c, q, Hq, 1)
    check(pu.attend(c, q, Hq, 1), ref, bound, (bits, D))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_one_step_in_two_calls(bits):
    """A step's single tokens and its chunk in a call each, on parts of the same arrays: the tokens' rows lie first, so
    that their call's T ends with them, and the chunk's call takes the last sequence's entries."""
    D, Hq, Hkv, page = 128, 8, 2, 32
    seqs = [(1, 900), (1, 64), (1, 1), (1, 1500), (100, 700)]
    c = pu.Cache(seqs, Hkv, D, page, bits, 3)
    c.fill(11)
    whole = pu.Cache(seqs, Hkv, D, page, bits, 3)
    whole.fill(11)
    x = pu.normal((c.N, Hq + 2 * Hkv, D), 5)
    rope = pu.rope_table(1500, D)
    W, k = (Hq + 2 * Hkv) * D, len(seqs) - 1
    q_ref = np.empty((c.N, Hq, D), np.uint16)
    for b, (n, kv) in enumerate(seqs):
        r, pos = slice(c.start[b], c.start[b + 1]), np.arange(kv - n, kv)
        q_ref[r] = pu.rotate(x[r, :Hq], pos, rope, D, 0)
        whole.put(b, kv - n, pu.rotate(x[r, Hq:Hq + Hkv], pos, rope, D, 0), x[r, Hq + Hkv:])
    with ts.DeviceBuffer.from_array(x) as dx, ts.DeviceBuffer(c.N * Hq * D * 2) as do, \
            ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds, ts.DeviceBuffer.from_array(rope) as dr:
        do.fill_bytes(0xFF)
        first = c.device()
        d = c.bufs
        ks, vs = (d["ks"], d["vs"]) if bits == 4 else (None, None)
        first.B = k
        last = ts.KvCache(d["k"], d["v"], d["table"].ptr + 4 * k * c.cols, d["kv_len"].ptr + 4 * k,
                          d["start"].ptr + 4 * k, 1, c.cols, c.pages, page, Hkv, D, bits, ks, vs)
        q, kk, v = (ts.Rows(dx.ptr + 2 * D * h, W, D) for h in (0, Hq, Hq + Hkv))
        o = ts.Rows(do, Hq * D, D)
        for desc, T, mq, mkv in ((first, k, 1, 1500), (last, c.N, 100, 700)):
            ts.attn_kv_append(desc, q, q, kk, v, T, Hq, dr, len(rope), D, 0, mq)
            ts.attn_paged(desc, q, o, T, Hq, 1, None, mq, mkv, ds)
        ts.synchronize()
        got_q = dx.download(np.uint16).reshape(x.shape)[:, :Hq]
        O = pu.f32(do.download(np.uint16)).reshape(c.N, Hq, D)
    c.download()
    assert np.array_equal(got_q, q_ref)
    for y in ("k", "v", "ks", "vs"):
        assert np.array_equal(getattr(c, y), getattr(whole, y)), y
    ref, bound = pu.attend_ref(c, q_ref, Hq, 1)
    check(O, ref, bound, bits)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n", [1, 8, 40])
def test_shared_pages(bits, n):
    """Sequences that share the pages of a prefix, one of them a page twice."""
    D, Hq, Hkv, page = 64, 8, 2, 16
    c = pu.Cache([(n, 300), (n, 210), (n, 500)], Hkv, D, page, bits, 3)
    c.fill(11)
    c.table[1, :12] = c.table[0, :12]
    c.table[2, 20] = c.table[2, 3]
    q = pu.normal((c.N, Hq, D), 5)
    ref, bound = pu.attend_ref(c, q, Hq, 1)
    check(pu.attend(c, q, Hq, 1), ref, bound, (bits, n))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_graph_of_a_chunk_replayed_with_other_lengths(bits):
    """A captured step of up to 64 tokens a sequence (append, attend in prefill tiles, read back), replayed with other
    tokens, starts, lengths and pages, none among them, each time against the same step run eagerly."""
    D, Hq, Hkv, page, cols, T = 128, 8, 2, 16, 60, 140
    hip = pu.Hip()
    c = pu.Cache([(1, cols * page)] * 3, Hkv, D, page, bits, 3, spare=0, cols=cols)
    c.fill(5)
    desc = c.device()
    clean = {y: getattr(c, y).copy() for y in ("k", "v", "ks", "vs")}
    rope, W = pu.rope_table(cols * page, D), (Hq + 2 * Hkv) * D
    with ts.DeviceBuffer(T * W * 2) as dx, ts.DeviceBuffer(T * Hq * D * 2) as dq, \
            ts.DeviceBuffer(T * Hq * D * 2) as do, ts.DeviceBuffer(2 * T * Hkv * D * 2) as dk, \
            ts.DeviceBuffer.from_array(rope) as dr, ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds:
        q, qo, o = ts.Rows(dx, W, D), ts.Rows(dq, Hq * D, D), ts.Rows(do, Hq * D, D)
        k, v = (ts.Rows(dx.ptr + 2 * D * h, W, D) for h in (Hq, Hq + Hkv))
        bk, bv = ts.Rows(dk, 2 * Hkv * D, D), ts.Rows(dk.ptr + 2 * Hkv * D, 2 * Hkv * D, D)
        plan = ts.attn_paged_plan(desc, T, Hq, 1, None, 64, cols * page)
        assert "prefill" in plan[0][0] and len(plan) == 2, plan

        def step():
            ts.attn_kv_append(desc, q, qo, k, v, T, Hq, dr, len(rope), D, 0, 64)
            ts.attn_paged(desc, qo, o, T, Hq, 1, None, 64, cols * page, ds)
            ts.attn_kv_read(desc, bk, bv, T, 64)

        st = hip.stream()
        ex = hip.capture(st, step)
        for it, seqs in enumerate([[(64, 64), (1, 400), (30, 960)], [(0, 17), (64, 700), (64, 65)],
                                   [(1, 1), (1, 2), (1, 959)], [(0, 0), (0, 0), (0, 0)], [(10, 200), (0, 9), (64, 64)]]):
            c.seqs, c.kv_len = seqs, np.array([x for _, x in seqs], np.int32)
            c.start = np.concatenate([[0], np.cumsum([x for x, _ in seqs])]).astype(np.int32)
            c.N = int(c.start[-1])
            c.table = np.random.default_rng(it).permutation(c.pages)[:3 * cols].astype(np.int32).reshape(3, cols)
            got = []
            for run in (lambda: hip("hipGraphLaunch", ex, st), step):
                for y in clean:
                    setattr(c, y, clean[y].copy())
                c.device()
                dx.upload(pu.normal((T, Hq + 2 * Hkv, D), 40 + it))
                for d in (dq, do, dk):
                    d.fill_bytes(0xFF)
                ts.synchronize()
                run()
                ts.synchronize()
                c.download()
                got.append([d.download(np.uint16) for d in (do, dq, dk)] + [getattr(c, y).copy() for y in clean])
            for a, b in zip(*got):
                assert np.array_equal(a, b), it
            O = got[0][0].reshape(T, Hq, D)
            assert np.all(O[c.N:] == 0xFFFF)
            if c.N:
                ref, bound = pu.attend_ref(c, got[0][1].reshape(T, Hq, D)[:c.N], Hq, 1)
                check(pu.f32(O[:c.N]), ref, bound, it)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Hq", [4, 128])
def test_rows_past_4_gib(bits, Hq):
    """Token tensors whose rows lie 2 GiB apart, by tokens and then by heads."""
    D, Hkv, page, n, kv = 64, 4, 32, 3, 600
    far = (1 << 30) + 8
    H = Hq + 2 * Hkv
    c = pu.Cache([(n, kv)], Hkv, D, page, bits, 3)
    c.fill(11)
    rope = pu.rope_table(kv, D)
    x = pu.normal((n, H, D), 5)
    with ts.DeviceBuffer(3 * 2 * far + (1 << 20)) as big, ts.DeviceBuffer.from_array(rope) as dr, \
            ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds, \
            ts.DeviceBuffer(n * Hq * D * 2) as near:
        for i in range(n):
            pu.memcpy_to(big.ptr + 2 * i * far, x[i])

        def rows(h):
            return ts.Rows(big.ptr + 2 * D * h, far, D)

        desc = c.device()
        ts.attn_kv_append(desc, rows(0), rows(0), rows(Hq), rows(Hq + Hkv), n, Hq, dr, kv, D, 0, n)
        ts.attn_paged(desc, rows(0), rows(H), n, Hq, 1, None, n, kv, ds)
        ts.attn_kv_read(desc, rows(2 * H), rows(2 * H + Hkv), n, n)
        ts.attn_paged(desc, rows(0), ts.Rows(near, Hq * D, D), n, Hq, 1, None, n, kv, ds)
        ts.synchronize()
        got = np.stack([memcpy_from(big.ptr + 2 * i * far, (4 * H, D)) for i in range(n)])
        same = near.download(np.uint16).reshape(n, Hq, D)
        c.download()
        pos = np.arange(kv - n, kv)
        q = pu.rotate(x[:, :Hq], pos, rope, D, 0)
        assert np.array_equal(got[:, :Hq], q)
        ref, bound = pu.attend_ref(c, q, Hq, 1)
        check(pu.f32(got[:, H:H + Hq]), ref, bound, (bits, Hq))
        assert np.array_equal(got[:, H:H + Hq], same)
        K, V = c.get(0, kv - n, kv)
        assert np.array_equal(pu.f32(got[:, 2 * H:2 * H + Hkv]), K)
        assert np.array_equal(pu.f32(got[:, 2 * H + Hkv:2 * H + 2 * Hkv]), V)
        # heads apart: three of them, one kv head
        if bits == 16 and Hq == 4:
            d = pu.Cache([(n, kv)], 1, D, page, bits, 3)
            d.fill(12)
            y = pu.normal((n, 3, D), 6)
            for h in range(3):
                pu.memcpy_to(big.ptr + 2 * h * far, np.ascontiguousarray(y[:, h]))
            ts.attn_paged(d.device(), ts.Rows(big, D, far), ts.Rows(big.ptr + 4096, D, far), n, 3, 1, None, n, kv, ds)
            ts.synchronize()
            O = np.stack([memcpy_from(big.ptr + 4096 + 2 * h * far, (n, D)) for h in range(3)], 1)
            ref, bound = pu.attend_ref(d, y, 3, 1)
            check(pu.f32(O), ref, bound, "heads")


@pytest.mark.gpu
@pytest.mark.parametrize("bits,D,n", [(16, 16, 1), (4, 64, 1), (16, 16, 9), (16, 16, 20), (4, 64, 30)])
def test_the_longest_sequence(bits, D, n):
    """2^30 keys in a table row whose entries name a few pages over and over, and one page once, at the very end, which
    holds the keys that the rows look for: one that all of them see, and the last of all, which the last row sees.
    These outweigh each other key by e^39, and there are e^20.8 of those, so that what they add is lost in the
    roundings: 2^-8 each of P and O, and 2^-8 for the scores', of a magnitude of 40 and D + 16 times 2^-24 each."""
    page, cols, Hkv, Hq = 256, 1 << 22, 1, 4
    c = pu.Cache([(n, 8 * page)], Hkv, D, page, bits, 3, spare=0, cols=8)
    K, V = pu.normal((8 * page, Hkv, D), 1, 0.01), pu.normal((8 * page, Hkv, D), 2)
    K[-1], K[-n - 1] = 0x3F80, 0x3F80  # ones: the last key of all, and one that every row sees
    c.put(0, 0, K, V)
    held = c.get(0, 0, 8 * page)
    table = np.empty((1, cols), np.int32)
    table[0] = c.table[0, np.arange(cols) % 7]
    table[0, -1] = c.table[0, 7]
    q = np.full((n, Hq, D), pu.bf16(np.float32(40.0 / D ** 0.5)), np.uint16)  # a score of 40 with a key of ones
    base = c.device()
    with ts.DeviceBuffer.from_array(table) as dt, ts.DeviceBuffer.from_array(np.array([1 << 30], np.int32)) as dl, \
            ts.DeviceBuffer.from_array(q) as dq, ts.DeviceBuffer(q.nbytes) as do, \
            ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds:
        do.fill_bytes(0xFF)
        desc = ts.KvCache(c.bufs["k"], c.bufs["v"], dt, dl, base.q_start, 1, cols, 8, page, Hkv, D, bits,
                          c.bufs["ks"] if bits == 4 else None, c.bufs["vs"] if bits == 4 else None)
        ts.attn_paged(desc, ts.Rows(dq, Hq * D, D), ts.Rows(do, Hq * D, D), n, Hq, 1, None, n, 1 << 30, ds)
        ts.synchronize()
        O = pu.f32(do.download(np.uint16)).reshape(n, Hq, D)
    times = np.array([(cols - 1) // 7 + (p < (cols - 1) % 7) for p in range(7)] + [1], np.float64)
    count = np.repeat(times, page)
    x = pu.f32(q[0, 0]).astype(np.float64)
    s = D ** -0.5 * (held[0][:, 0] @ x)
    for i in range(n):
        w = count * np.exp(s - 40.0)
        w[8 * page - (n - 1 - i):] = 0  # keys behind the row's position
        w /= w.sum()
        ref, A = w @ held[1][:, 0], w @ np.abs(held[1][:, 0])
        assert w[-n - 1] > 0.4, w[-n - 1]
        bound = 2.0 ** -8 * np.abs(ref) + A * 2.0 ** -8 * 1.01 + 2.0 ** -8 * A
        assert np.all(np.abs(O[i] - ref) <= bound), (i, float(np.abs(O[i] - ref).max()))


@pytest.mark.gpu
def test_every_code_under_every_scale():
    """A cache that another program wrote: 16 codes in both halves of a byte under all 256 scale bytes read as
    code times 2^(e - 127) to the last bit, below bf16's normal numbers too, as infinities past its range and as NaN
    under 255."""
    D, page = 64, 256
    c = pu.Cache([(page, page)], 1, D, page, 4, 1, spare=0)
    low = np.arange(32) % 16
    c.k[0, 0] = np.tile((low | (low[::-1] << 4)).astype(np.uint8), (page, 1))
    c.v[0, 0] = np.tile((low[::-1] | (low << 4)).astype(np.uint8), (page, 1))
    c.ks[0, 0] = np.stack([np.arange(256), np.arange(256)[::-1]], 1)
    c.vs[0, 0] = c.ks[0, 0, ::-1]
    with ts.DeviceBuffer(page * D * 2) as dk, ts.DeviceBuffer(page * D * 2) as dv:
        ts.attn_kv_read(c.device(), ts.Rows(dk, D, D), ts.Rows(dv, D, D), page, page)
        ts.synchronize()
        got = [pu.f32(d.download(np.uint16)).astype(np.float64).reshape(page, D) for d in (dk, dv)]
    for x, want in zip(got, c.get(0, 0, page)):
        want = want[:, 0]
        want = np.where(np.abs(want) >= 2.0 ** 128, np.copysign(np.inf, want), want)
        assert np.isinf(want).any() and np.isnan(want).any() and (np.abs(want) < 2.0 ** -127).any()
        assert np.array_equal(x, want, equal_nan=True)
