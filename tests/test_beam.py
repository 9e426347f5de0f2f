"""Beam search's selection and the cache's reordering on the GPU, against their definitions in numpy."""
import numpy as np
import pytest

import paged_util as pu
import transfer_station_amd as ts
from paged_util import bf16, f32

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module", autouse=True)
def _gpu_present():
    assert ts.device_count() >= 1, "no HIP device visible: GPU tests must run on the MI355X box"


# ---- selection --------------------------------------------------------------------------------
def select_ref(x, scores, done, done_token, B, beams, K):
    """x float64 [rows][V]. (score, token, parent), and each score's log-sum-exp."""
    V = x.shape[1]
    out = np.full((B, K), -np.inf), np.full((B, K), -1), np.repeat(beams * np.arange(B)[:, None], K, 1)
    for b in range(B):
        rows = slice(b * beams, (b + 1) * beams)
        # [beam][its continuations, by logit and token]: a stable sort by score then has the order of ties.
        c, tok = np.full((beams, min(K, V)), -np.inf), np.zeros((beams, min(K, V)), int)
        for i, r in enumerate(range(rows.start, rows.stop)):
            if not np.isfinite(scores[r]):
                continue
            if done is not None and done[r]:
                c[i, 0], tok[i, 0] = scores[r], done_token
            elif np.all(np.isfinite(x[r]) | (x[r] == -np.inf)) and np.any(np.isfinite(x[r])):
                top = x[r].max()
                tok[i] = np.argsort(-x[r], kind="stable")[:K]
                c[i] = (x[r, tok[i]] - (top + np.log(np.exp(x[r] - top).sum()))) + float(scores[r])
        best = np.argsort(-c.reshape(-1), kind="stable")[:K]
        best = best[np.isfinite(c.reshape(-1)[best])]
        out[0][b, :len(best)], out[1][b, :len(best)] = c.reshape(-1)[best], tok.reshape(-1)[best]
        out[2][b, :len(best)] = b * beams + best // c.shape[1]
    return out


def select(logits, scores, done, done_token, B, beams, V, K, shift=0):
    """logits [rows][row stride], uint16 or float32, starting `shift` elements into their buffer."""
    size = logits.itemsize
    raw = np.concatenate([np.zeros(shift, logits.dtype), logits.ravel()])
    with ts.DeviceBuffer.from_array(raw) as dl, ts.DeviceBuffer.from_array(scores) as dsc, \
            ts.DeviceBuffer.from_array(done if done is not None else np.zeros(1, np.uint8)) as dd, \
            ts.DeviceBuffer(4 * B * K + 4) as o0, ts.DeviceBuffer(4 * B * K + 4) as o1, \
            ts.DeviceBuffer(4 * B * K + 4) as o2:
        call = ts.Beams(dl.ptr + size * shift, logits.shape[1], 8 * size, B, beams, V, K, dsc,
                        dd if done is not None else None, done_token)
        with ts.DeviceBuffer(ts.attn_beam_scratch_bytes(call)) as s:
            for x in (o0, o1, o2, s):
                x.fill_bytes(0xFF)
            ts.attn_beam_select(call, o0, o1, o2, s)
            ts.synchronize()
            got = [o.download(np.uint32) for o in (o0, o1, o2)]
    assert all(g[-1] == 0xFFFFFFFF for g in got)
    return (got[0][:-1].view(np.float32).reshape(B, K), got[1][:-1].view(np.int32).reshape(B, K),
            got[2][:-1].view(np.int32).reshape(B, K))


def check_select(got, ref):
    # The sums of exponentials in fp32: each off by 2^-20 at most, as is their sum; the score is rounded once.
    want = ref[0]
    fine = np.isfinite(want)
    assert np.array_equal(got[0][~fine], want[~fine])
    assert np.all(np.abs(got[0][fine] - want[fine]) <= 2.0 ** -24 * np.abs(want[fine]) + 2.0 ** -19)
    assert np.array_equal(got[1], ref[1]) and np.array_equal(got[2], ref[2])


def logits_of(rows, V, bits, seed, sigma=2.5, extra=0):
    x = pu.normal((rows, V + extra), seed, sigma)
    return x if bits == 16 else f32(x) + f32(pu.normal((rows, V + extra), seed + 1, 0.01))


def as64(x):
    return (f32(x) if x.dtype == np.uint16 else x).astype(np.float64)


# (B, beams, V, K, bits, extra elements between rows, shift of the first)
SELECT = [
    (1, 1, 1, 1, 32, 0, 0), (1, 4, 7, 8, 16, 0, 1), (2, 3, 50257, 6, 32, 0, 0), (3, 4, 50257, 8, 16, 0, 1),
    (2, 5, 8192, 64, 16, 0, 0), (1, 16, 2049, 33, 32, 3, 1), (40, 8, 32001, 16, 16, 7, 0),
    (1, 256, 100, 64, 16, 0, 0), (1, 2, 262147, 4, 32, 0, 0), (2, 1, 5, 20, 32, 0, 0), (300, 4, 9000, 8, 32, 0, 0),
    (1, 3, 1 << 20, 7, 16, 0, 0), (1, 13, 238968, 13, 16, 0, 0), (4, 64, 32000, 64, 32, 0, 0), (1, 200, 40000, 64, 16, 0, 0),
    (2, 256, 5000, 50, 16, 0, 0), (1, 5, 120000, 64, 32, 0, 0),
]


@pytest.mark.parametrize("case", range(len(SELECT)))
def test_select(case):
    B, beams, V, K, bits, extra, shift = SELECT[case]
    say("select", SELECT[case])
    x = logits_of(B * beams, V, bits, 10 * case, extra=extra)
    scores = -np.sort(np.random.default_rng(case).random(B * beams) * 9).astype(np.float32)
    ref = select_ref(as64(x)[:, :V], scores, None, 0, B, beams, K)
    check_select(select(x, scores, None, 0, B, beams, V, K, shift), ref)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("V", [700, 30011])
def test_select_ties_masks_and_done_beams(V, bits):
    """Equal logits in all places, rows with few or no logits left, complete and impossible beams."""
    say("select ties", V, bits)
    B, beams, K = 6, 4, 12
    rng = np.random.default_rng(V + bits)
    x = np.round(rng.standard_normal((B * beams, V)) * 2).astype(np.float32)  # few values: ties everywhere
    x[4] = 1.5                                  # all equal
    x[5] = -np.inf                              # nothing left
    x[6, 3:] = -np.inf                          # three left
    x[8:12] = 0.0                               # an entry of equal rows
    x[13, rng.integers(0, V, V // 2)] = -np.inf
    x[14, 11] = np.nan
    x[15, 12] = np.inf
    x[16:20] = -np.inf                          # an entry with nothing but a complete beam
    x[20:24, 5:] = -np.inf
    scores = (-rng.random(B * beams) * 5).astype(np.float32)
    scores[8:12] = -1.0
    scores[12] = -np.inf
    scores[21] = np.nan
    scores[22] = np.inf
    done = np.zeros(B * beams, np.uint8)
    done[[1, 9, 18]] = 1
    logits = bf16(x) if bits == 16 else x
    ref = select_ref(x.astype(np.float64), scores, done, 2, B, beams, K)
    check_select(select(logits, scores, done, 2, B, beams, V, K), ref)


def test_select_more_equal_logits_than_there_is_room_for():
    """Every chunk of every row holds thousands of logits of the largest value."""
    B, beams, V, K = 1, 32, 40000, 64
    x = np.zeros((beams, V), np.float32)
    x[:, 17::3] = 4.0
    x[3, 9000:9010] = 5.0
    scores = np.full(beams, -2.0, np.float32)
    check_select(select(bf16(x), scores, None, 0, B, beams, V, K), select_ref(x.astype(np.float64), scores, None, 0,
                                                                             B, beams, K))


def test_select_ascending_logits():
    """The largest logits in a few threads' hands: all of a chunk's best lie side by side."""
    for V, K in ((20000, 64), (8192, 33)):
        x = np.sort(np.random.default_rng(V).standard_normal((2, V)).astype(np.float32), 1)
        scores = np.zeros(2, np.float32)
        check_select(select(x, scores, None, 0, 1, 2, V, K), select_ref(x.astype(np.float64), scores, None, 0, 1, 2, K))


# ---- reordering -------------------------------------------------------------------------------
class Pool:
    """Groups of beams over a paged cache: pages of the prompt are shared, those behind it own; bytes are random."""

    def __init__(self, lens, beams, shared, cols, Hkv, D, page, bits, seed):
        rng = np.random.default_rng(seed)
        self.beams, self.cols, self.Hkv, self.D, self.page, self.bits = beams, cols, Hkv, D, page, bits
        G, B = len(lens), len(lens) * beams
        self.B, self.pages = B, G * shared + B * (cols - shared) + 2
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.zeros((B, cols), np.int32)
        for b in range(B):
            for j in range(cols):
                self.table[b, j] = order[b // beams * shared + j if j < shared
                                         else G * shared + b * (cols - shared) + j - shared]
        self.lens = np.repeat(np.array(lens, np.int32), beams)
        rb = 2 * D if bits == 16 else D // 2
        self.data = {x: rng.integers(0, 256, (self.pages, Hkv, page, rb), np.uint8) for x in "kv"}
        if bits == 4:
            self.data.update({x + "s": rng.integers(0, 256, (self.pages, Hkv, page, D // 32), np.uint8)
                              for x in "kv"})

    def expect(self, parent, tables=1):
        """(table, data, which bytes are set) once the sequences have followed their parents."""
        table, data = self.table.copy(), {x: a.copy() for x, a in self.data.items()}
        free = {x: np.zeros(a.shape, bool) for x, a in self.data.items()}
        for b in range(self.B):
            first = b // self.beams * self.beams
            p = parent[b] if first <= parent[b] < first + self.beams else b
            n = min(max(int(self.lens[first]), 0), self.cols * self.page)
            full, rest = divmod(n, self.page)
            if tables:
                table[b, :full] = self.table[p, :full]
            if rest and p != b and 0 <= self.table[p, full] < self.pages and 0 <= self.table[b, full] < self.pages:
                for x, a in data.items():
                    a[self.table[b, full], :, :rest] = self.data[x][self.table[p, full], :, :rest]
                    # Up to 16 bytes may be copied whole.
                    end = -(-rest * a.shape[-1] // 16) * 16 // a.shape[-1]
                    free[x][self.table[b, full], :, rest:end] = True
        return table, data, free

    def run(self, parent, tables=1):
        bufs = {x: ts.DeviceBuffer.from_array(a) for x, a in self.data.items()}
        with ts.DeviceBuffer.from_array(self.table) as dt, ts.DeviceBuffer.from_array(self.lens) as dl, \
                ts.DeviceBuffer.from_array(np.asarray(parent, np.int32)) as dp:
            c = ts.KvCache(bufs["k"], bufs["v"], dt, dl, dl, self.B, self.cols, self.pages, self.page, self.Hkv, self.D,
                           self.bits, bufs.get("ks"), bufs.get("vs"))
            ts.attn_kv_reorder(c, dp, self.beams, tables)
            ts.synchronize()
            got = dt.download(np.int32).reshape(self.table.shape), {
                x: b.download(np.uint8).reshape(self.data[x].shape) for x, b in bufs.items()}
        for b in bufs.values():
            b.free()
        return got

    def check(self, parent, tables=1):
        want, got = self.expect(parent, tables), self.run(parent, tables)
        assert np.array_equal(got[0], want[0])
        for x in self.data:
            same = (got[1][x] == want[1][x]) | want[2][x]
            assert np.all(same), (x, np.argwhere(~same)[:5])


# (lengths of the groups, beams, shared pages, columns, Hkv, D, page, bits)
REORDER = [
    ([5], 1, 0, 1, 1, 16, 16, 16), ([77, 64, 65, 0], 4, 2, 6, 2, 64, 32, 16), ([33], 4, 1, 3, 8, 128, 16, 16),
    ([40, 47], 5, 0, 4, 3, 80, 16, 16), ([100, 127, 128], 8, 1, 3, 2, 256, 64, 16), ([61], 32, 2, 5, 1, 48, 16, 16),
    ([77, 64, 63], 4, 2, 6, 2, 64, 32, 4), ([130, 1], 12, 0, 3, 2, 128, 64, 4), ([300], 20, 1, 3, 1, 256, 128, 4),
    ([255, 7], 3, 0, 2, 16, 128, 256, 4),
]


@pytest.mark.parametrize("case", range(len(REORDER)))
def test_reorder(case):
    say("reorder", REORDER[case])
    lens, beams = REORDER[case][:2]
    p = Pool(*REORDER[case], seed=case)
    rng = np.random.default_rng(50 + case)
    first = np.repeat(beams * np.arange(len(lens)), beams)
    p.check(first + rng.integers(0, beams, p.B))          # any parents
    p.check(first + (np.arange(p.B) - first + 1) % beams)  # a cycle: everyone moves, nobody is lost
    p.check(first)                                         # all follow the first
    p.check(np.arange(p.B), 1)                             # nothing moves
    p.check(first + rng.integers(0, beams, p.B), 0)        # another layer's cache


def test_reorder_bad_entries():
    """Parents outside the group, pages outside the cache, lengths outside the table."""
    p = Pool([37, 5, 2 ** 31 - 1, -4], 4, 0, 4, 2, 64, 16, 16, seed=9)
    p.table[1, 2], p.table[6, 0] = -1, 10 ** 6
    p.check(np.array([3, 0, 1, -1, 2 ** 31 - 1, 6, 4, 5, 9, 8, 0, 10, 12, 15, 13, -2 ** 31], np.int64).astype(np.int32))
