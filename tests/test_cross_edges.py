"""Cross attention on the GPU where it can go wrong: layouts, starts and lengths of any kind, bounds that do not hold, far
offsets, sharp rows, NaN in places of others, graphs and streams."""
import numpy as np
import pytest

import cross_util as cu
import paged_util as pu
import transfer_station_amd as ts
from paged_util import f32
from transfer_station_amd import _lib

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module", autouse=True)
def _gpu_present():
    assert ts.device_count() >= 1, "no HIP device visible: GPU tests must run on the MI355X box"


SHAPES = [([(1, 700), (3, 90)], 8, 4, 64), ([(140, 200), (37, 65)], 4, 2, 128)]


@pytest.mark.parametrize("shape", range(2))
@pytest.mark.parametrize("max_q,max_k", [(1, 1), (5, 64), (100000, 100000), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_bounds_that_do_not_hold(shape, max_q, max_k):
    say("bounds", shape, max_q, max_k)
    t = cu.Batch(*SHAPES[shape], 7)
    cu.check(t, cu.run(t, max_q=max_q, max_k=max_k), cu.reference(t))


@pytest.mark.parametrize("shape", range(2))
def test_rows_wider_than_their_heads(shape):
    t = cu.Batch(*SHAPES[shape], 8, stride=24)
    cu.check(t, cu.run(t), cu.reference(t))


@pytest.mark.parametrize("shape", range(2))
def test_the_same_call_gives_the_same_bits(shape):
    t = cu.Batch(*SHAPES[shape], 9)
    a, b = cu.run(t), cu.run(t)
    assert all(np.array_equal(a[x].view(np.uint32), b[x].view(np.uint32)) for x in a)


@pytest.mark.parametrize("sigma,scale", [(30.0, 0.0), (1.0, 3.0), (1.0, 1e-4), (300.0, 0.0)])
@pytest.mark.parametrize("shape", range(2))
def test_sharp_and_flat_rows(shape, sigma, scale):
    say("sharp", shape, sigma, scale)
    t = cu.Batch(*SHAPES[shape], 10, sigma_q=sigma)
    cu.check(t, cu.run(t, scale=scale), cu.reference(t, scale))


@pytest.mark.parametrize("shape", range(2))
def test_without_the_log_sum_exp(shape):
    t = cu.Batch(*SHAPES[shape], 11)
    cu.check(t, cu.run(t, grad=False, lse=False), {"o": cu.reference(t, grad=False)["o"]})


class Call:
    """A call with its buffers: rows gives each tensor's array, first element and strides."""

    def __init__(self, t, arrays, rows):
        self.t, self.bufs = t, {}
        self.call = cu.call_of(t, self.bufs)
        for x, a in arrays.items():
            self.bufs[x] = ts.DeviceBuffer.from_array(a)
        self.rows = {x: ts.Rows(self.bufs[b].ptr + 2 * at, tok, head) for x, (b, at, tok, head) in rows.items()}
        self.bufs["lse"] = ts.DeviceBuffer(4 * t.Tq * t.Hq)
        self.bufs["s"] = ts.DeviceBuffer(ts.attn_cross_scratch_bytes(self.call))
        self.bufs["gs"] = ts.DeviceBuffer(ts.attn_cross_grad_scratch_bytes(self.call))

    def __call__(self, grad=True):
        r, b = self.rows, self.bufs
        ts.attn_cross(self.call, r["q"], r["k"], r["v"], r["o"], b["lse"], b["s"])
        if grad:
            ts.attn_cross_grad(self.call, r["q"], r["k"], r["v"], r["o"], b["lse"], r["go"], r["dq"], r["dk"], r["dv"],
                               b["gs"])

    def fill(self, *names):
        for x in names:
            self.bufs[x].fill_bytes(0xFF)


def plain(t):
    """The arrays and rows of a batch as they are."""
    arrays = {x: getattr(t, x) for x in ("q", "k", "v", "go")}
    arrays.update(o=np.full_like(t.q, 0xFFFF), dq=np.full_like(t.q, 0xFFFF), dk=np.full_like(t.k, 0xFFFF),
                  dv=np.full_like(t.k, 0xFFFF))
    return arrays, {x: (x, 0, a.shape[1], t.D) for x, a in arrays.items()}


def results(c):
    t, out = c.t, {}
    for x, heads in (("o", t.Hq), ("dq", t.Hq), ("dk", t.Hkv), ("dv", t.Hkv)):
        raw = c.bufs[x].download(np.uint16).reshape(-1, heads * t.D)
        out[x] = f32(raw).reshape(-1, heads, t.D)
    out["lse"] = c.bufs["lse"].download(np.float32).reshape(t.Tq, t.Hq)
    return out


@pytest.mark.parametrize("shape", range(2))
def test_heads_of_one_projection_and_head_major_rows(shape):
    """K, V, dK and dV as heads of one tensor [T][2 Hkv][D]; Q and its gradient head by head, [Hq][T][D]."""
    t = cu.Batch(*SHAPES[shape], 12)
    D, w = t.D, 2 * t.Hkv * t.D
    arrays, rows = plain(t)
    arrays["kv"] = np.concatenate([t.k, t.v], 1)
    arrays["dkv"] = np.full_like(arrays["kv"], 0xFFFF)
    qh = np.ascontiguousarray(t.q.reshape(t.Tq, t.Hq, D).transpose(1, 0, 2))
    arrays["q"], arrays["dq"] = qh, np.full_like(qh, 0xFFFF)
    rows.update(k=("kv", 0, w, D), v=("kv", w // 2, w, D), dk=("dkv", 0, w, D), dv=("dkv", w // 2, w, D),
                q=("q", 0, D, t.Tq * D), dq=("dq", 0, D, t.Tq * D))
    c = Call(t, arrays, rows)
    c()
    ts.synchronize()
    dkv = c.bufs["dkv"].download(np.uint16).reshape(-1, w)
    assert np.all(dkv[~t.live_k] == 0xFFFF)
    got = {"o": f32(c.bufs["o"].download(np.uint16)).reshape(-1, t.Hq, D),
           "dq": f32(c.bufs["dq"].download(np.uint16)).reshape(t.Hq, t.Tq, D).transpose(1, 0, 2),
           "dk": f32(dkv[:, :w // 2]).reshape(-1, t.Hkv, D), "dv": f32(dkv[:, w // 2:]).reshape(-1, t.Hkv, D)}
    cu.check(t, got, cu.reference(t))


@pytest.mark.parametrize("shape", range(2))
def test_one_head_read_as_many(shape):
    """A head stride of 0 in what is only read: all kv heads have the first one's K, all heads the first one's dO."""
    t = cu.Batch(*SHAPES[shape], 21)
    D = t.D
    for x, heads in ((t.k, t.Hkv), (t.go, t.Hq)):
        for h in range(1, heads):
            x[:, h * D:(h + 1) * D] = x[:, :D]
    arrays, rows = plain(t)
    rows.update(k=("k", 0, t.k.shape[1], 0), go=("go", 0, t.go.shape[1], 0))
    c = Call(t, arrays, rows)
    c()
    ts.synchronize()
    cu.check(t, results(c), cu.reference(t))


def test_starts_and_lengths_of_any_kind():
    """What they name is cut to the tensors: the rest is left as it was, and nothing outside is read or written."""
    t = cu.Batch([(30, 50), (1, 20), (4, 3), (2, 100), (3, 40)], 4, 2, 64, 13, room=(30, 100))
    q_start, q_len, Tq = t.spans["q"]
    k_start, k_len, Tk = t.spans["k"]
    q_len[1], k_len[1] = -5, 2 ** 31 - 1                    # no rows
    q_len[2], k_len[2] = 4, -2 ** 31                        # no states
    q_start[3], q_len[3] = Tq - 2, 2 ** 31 - 1              # the last two rows
    k_start[3], k_len[3] = 2 ** 31 - 1, 7                   # past the end: none
    q_start[4], q_len[4], k_start[4], k_len[4] = -7, 3, -1, 40  # from 0 on: rows that sequence 0 has
    q_start[0] = 5
    seqs = [(30, 50), (0, 0), (4, 0), (2, 0), (3, 40)]
    q_at, k_at = [5, 0, int(q_start[2]), Tq - 2, 0], [int(k_start[0]), 0, 0, 0, 0]
    k_start[0] = k_at[0] = 60
    t.q[:], t.k[:], t.v[:] = (pu.normal(x.shape, 14 + i) for i, x in enumerate((t.q, t.k, t.v)))
    c = Call(t, *plain(t))
    c.call = cu.call_of(t, c.bufs, max_q=30, max_k=100)
    c.fill("lse")
    c(grad=False)
    ts.synchronize()
    got = results(c)
    live = np.zeros(Tq, bool)
    r = cu.Batch(seqs, 4, 2, 64, 13)
    for b, (n, m) in enumerate(seqs):
        rows, states = slice(q_at[b], q_at[b] + n), slice(k_at[b], k_at[b] + m)
        live[rows] = True
        r.q[r.rows(b)[0]] = t.q[rows]
        r.k[r.rows(b)[1]], r.v[r.rows(b)[1]] = t.k[states], t.v[states]
    ref = cu.reference(r, grad=False)
    out = {x: np.zeros((r.Tq,) + got[x].shape[1:], np.float32) for x in ("o", "lse")}
    for b, (n, _) in enumerate(seqs):
        for x in out:
            out[x][r.rows(b)[0]] = got[x][q_at[b]:q_at[b] + n]
    cu.check(r, out, ref)
    raw = c.bufs["o"].download(np.uint16).reshape(Tq, -1)
    assert np.all(raw[~live] == 0xFFFF)


def test_sequences_may_share_states():
    """Forward: four decoders over two inputs, one of them over a part of its states."""
    t = cu.Batch([(7, 90), (3, 90), (1, 40), (5, 61)], 4, 4, 64, 15, room=(7, 100))
    t.spans["k"][0][:4] = 0, 0, 50, 100
    t.live_k[:] = True
    t.k[:], t.v[:] = pu.normal(t.k.shape, 16), pu.normal(t.v.shape, 17)
    cu.check(t, cu.run(t, grad=False), cu.reference(t, grad=False))


def test_nan_and_infinities_stay_with_their_own():
    """A row of NaN, and an input with an infinite state, spoil what they are part of and nothing else."""
    t = cu.Batch([(40, 60), (50, 70), (1, 30)], 4, 2, 64, 18)
    t.q[7, :64] = 0x7FC0                       # head 0 of row 7
    rows, states = t.rows(1)
    t.k[states.start + 3, :64] = 0x7F80        # kv head 0 of sequence 1
    c = Call(t, *plain(t))
    c()
    ts.synchronize()
    got, ref = results(c), cu.reference(t)
    bad_q, bad_k = np.zeros((t.Tq, 4), bool), np.zeros((t.Tk, 2), bool)
    bad_q[7, 0] = True
    bad_q[rows, :2] = True
    bad_k[t.rows(0)[1], 0] = True              # gradients of what row 7 has seen
    bad_k[states, 0] = True
    for x in ("o", "dq", "dk", "dv"):
        bad, live = (bad_q, t.live_q) if x in ("o", "dq") else (bad_k, t.live_k)
        ok = live[:, None] & ~bad
        assert np.all(np.abs(got[x] - ref[x][0])[ok] <= ref[x][1][ok]), x
    assert np.all(np.isnan(got["o"][7, 0])) and np.all(np.isnan(got["o"][rows, 0]).any(-1))


@pytest.mark.parametrize("seqs,D", [([(3, 600)], 128), ([(540, 520)], 64)])
def test_rows_megabytes_apart(seqs, D):
    """Token strides of 2^22 elements: 520 states are 4.4 GB of addresses, past what 32 bits hold."""
    say("far", seqs, D)
    t = cu.Batch(seqs, 2, 1, D, 19, pad=0)
    tok = ts.ATTN_TOKEN_MAX
    far = {x: (t.Tq, 2) for x in ("q", "go", "o", "dq")}
    far.update({x: (t.Tk, 1) for x in ("k", "v", "dk", "dv")})
    bufs = {x: ts.DeviceBuffer(2 * tok * (T - 1) + 2 * heads * D) for x, (T, heads) in far.items()}
    for x in ("q", "go", "k", "v"):
        for i, row in enumerate(getattr(t, x)):
            pu.memcpy_to(bufs[x].ptr + 2 * tok * i, row)
    small = {}
    call = cu.call_of(t, small)
    for x, n in (("lse", 4 * t.Tq * 2), ("s", ts.attn_cross_scratch_bytes(call)),
                 ("gs", ts.attn_cross_grad_scratch_bytes(call))):
        small[x] = ts.DeviceBuffer(n)
    r = {x: ts.Rows(bufs[x], tok, D) for x in far}
    ts.attn_cross(call, r["q"], r["k"], r["v"], r["o"], small["lse"], small["s"])
    ts.attn_cross_grad(call, r["q"], r["k"], r["v"], r["o"], small["lse"], r["go"], r["dq"], r["dk"], r["dv"],
                       small["gs"])
    ts.synchronize()
    got = {}
    for x in ("o", "dq", "dk", "dv"):
        T, heads = far[x]
        row = np.empty(heads * D, np.uint16)
        got[x] = np.zeros((T, heads, D), np.float32)
        for i in range(T):
            _lib.check(_lib.lib().attn_dev_memcpy_dtoh(row.ctypes.data, bufs[x].ptr + 2 * tok * i, row.nbytes), "copy")
            got[x][i] = f32(row).reshape(heads, D)
    for b in list(bufs.values()) + list(small.values()):
        b.free()
    cu.check(t, got, cu.reference(t))


@pytest.mark.parametrize("shape", range(2))
def test_a_captured_step_replayed_with_other_lengths(shape):
    """One graph of a forward and a backward call, replayed as the batch changes, with eager calls between."""
    seqs, Hq, Hkv, D = SHAPES[shape]
    room = (max(s[0] for s in seqs), max(s[1] for s in seqs))
    t = cu.Batch(seqs, Hq, Hkv, D, 20, room=room)
    c = Call(t, *plain(t))
    hip = pu.Hip()
    stream = hip.stream()
    c()
    ts.synchronize()
    ex = hip.capture(stream, c)
    lengths = [seqs, [(room[0], 0), (1, room[1])], [(0, 5), (room[0], 1)], seqs, [(2, 64), (2, 65)]]
    for i, now in enumerate(lengths):
        u = cu.Batch(now, Hq, Hkv, D, 30 + i, room=room)
        for x in ("q", "k", "v", "go"):
            c.bufs[x].upload(getattr(u, x))
        c.bufs["q_len"].upload(u.spans["q"][1])
        c.bufs["k_len"].upload(u.spans["k"][1])
        ref = cu.reference(u)
        outs = []
        for eager in (0, 1, 0):
            c.fill("o", "dq", "dk", "dv", "lse")
            ts.synchronize()
            if eager:
                c()
            else:
                hip("hipGraphLaunch", ex, stream)
            ts.synchronize()
            outs.append(results(c))
        c.t = t
        for got in outs:
            cu.check(u, got, ref, "lengths %d" % i)
            assert all(np.array_equal(got[x].view(np.uint32), outs[0][x].view(np.uint32)) for x in got)


def test_two_streams_at_once():
    """Calls that overlap, each with workspaces of its own, give what they give alone."""
    ts_ = [cu.Batch([(300, 900)], 8, 4, 128, 40), cu.Batch([(2, 4000), (1, 100)], 16, 4, 64, 41)]
    calls = [Call(t, *plain(t)) for t in ts_]
    hip = pu.Hip()
    streams = [hip.stream(), hip.stream()]
    ts.synchronize()
    for _ in range(5):
        for c, s in zip(calls, streams):
            ts.set_stream(s.value)
            c()
    ts.set_stream(None)
    ts.synchronize()
    for c in calls:
        cu.check(c.t, results(c), cu.reference(c.t))
