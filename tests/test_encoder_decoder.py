"""An encoder-decoder's beam search on the GPU, token by token, as a server runs it: each layer appends the tokens to its
paged cache and attends to it and to the input's states; the beams that go on are chosen from the logits, and the caches
follow them. Each operator is checked against its definition on what it was given, and the caches against the tokens that
each beam really holds."""
import numpy as np
import pytest

import cross_util as cu
import paged_util as pu
import test_beam
import transfer_station_amd as ts
from paged_util import bf16, f32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu_present():
    assert ts.device_count() >= 1, "no HIP device visible: GPU tests must run on the MI355X box"


class Tokens:
    """What the beams hold, in the shape of a paged cache."""

    def __init__(self, layer, histories):
        self.layer, self.histories = layer, histories
        self.Hkv, self.D, self.B = layer.Hkv, layer.D, len(histories)
        self.seqs, self.start = [(1, len(h)) for h in histories], np.arange(self.B + 1)
        self.cols, self.page = 1 << 20, 1

    def get(self, b, lo, hi):
        h, out = self.histories[b][lo:hi], []
        for x in (self.layer.k[h], self.layer.v[h]):
            out.append(pu.values4(*pu.quantise(x)) if self.layer.bits == 4 else f32(x).astype(np.float64))
        return out


class Layer:
    """A token's q, k and v (rows of tables), the layer's pools, and the input's states."""

    def __init__(self, cache, V, Hq, states, bits, seed):
        self.Hq, self.Hkv, self.D, self.bits = Hq, cache.Hkv, cache.D, bits
        self.q, self.k, self.v = (pu.normal((V, h, self.D), seed + i)
                                  for i, h in enumerate((Hq, self.Hkv, self.Hkv)))
        self.pools = [ts.DeviceBuffer.from_array(getattr(cache, x)) for x in ("k", "v", "ks", "vs")]
        self.cache = cache
        self.states = states
        self.kv = ts.DeviceBuffer.from_array(np.concatenate([states.k, states.v], 1))
        self.ins = [ts.DeviceBuffer(2 * cache.B * h * self.D) for h in (Hq, self.Hkv, self.Hkv)]
        self.qr, self.o1, self.o2 = (ts.DeviceBuffer(2 * cache.B * Hq * self.D) for _ in range(3))

    def desc(self, c):
        d = ts.KvCache(self.pools[0], self.pools[1], c.bufs["table"], c.bufs["kv_len"], c.bufs["start"], c.B, c.cols,
                       c.pages, c.page, c.Hkv, c.D, self.bits, *(self.pools[2:] if self.bits == 4 else (None, None)))
        return d


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("bits,Hkv", [(16, 2), (4, 4)])
def test_beam_search(bits, Hkv, graph):
    G, beams, Hq, D, V, page, eos, steps = 3, 4, 4, 64, 1000, 16, 7, 24
    B, prompt = G * beams, [5, 31, 16]
    lens = np.repeat(prompt, beams)
    c = pu.Cache([(1, int(n) + steps) for n in lens], Hkv, D, page, bits, 1)
    c.kv_len = lens.astype(np.int32)
    c.device()
    seqs = [(beams, 90), (beams, 1), (beams, 333)]
    layers = []
    rng = np.random.default_rng(2)
    told = [rng.integers(0, V, n) for n in prompt]
    hist = [list(told[b // beams]) for b in range(B)]
    for i in range(2):
        c.k[:], c.v[:], c.ks[:], c.vs[:] = 0xFF, 0xFF, 0xFF, 0xFF
        layer = Layer.__new__(Layer)
        states = cu.Batch(seqs, Hq, Hkv, D, 20 + 10 * i)
        tables = [pu.normal((V, h, D), 50 + 3 * i + j) for j, h in enumerate((Hq, Hkv, Hkv))]
        for b in range(B):
            c.put(b, 0, tables[1][hist[b]], tables[2][hist[b]])
        layer.__init__(c, V, Hq, states, bits, 50 + 3 * i)
        layers.append(layer)
    small = {}
    W = np.random.default_rng(3).standard_normal((Hq * D, V)).astype(np.float32) * 0.15
    logits, scores = ts.DeviceBuffer(4 * B * V), ts.DeviceBuffer(4 * B)
    done, best = ts.DeviceBuffer(B), [ts.DeviceBuffer(4 * B) for _ in range(3)]
    call = cu.call_of(layers[0].states, small)
    select = ts.Beams(logits, V, 32, G, beams, V, beams, scores, done, eos)
    s1 = ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128))
    s2 = ts.DeviceBuffer(ts.attn_cross_scratch_bytes(call))
    s3 = ts.DeviceBuffer(ts.attn_beam_scratch_bytes(select))
    cap = max(prompt) + steps

    def attend():
        for y in layers:
            d, w, u = y.desc(c), Hq * D, Hkv * D
            ts.attn_kv_append(d, ts.Rows(y.ins[0], w, D), ts.Rows(y.qr, w, D), ts.Rows(y.ins[1], u, D),
                              ts.Rows(y.ins[2], u, D), B, Hq, None, 0, 0)
            ts.attn_paged(d, ts.Rows(y.qr, w, D), ts.Rows(y.o1, w, D), B, Hq, 1, None, 1, cap, s1)
            ts.attn_cross(call, ts.Rows(y.o1, w, D), ts.Rows(y.kv, 2 * u, D), ts.Rows(y.kv.ptr + 2 * u, 2 * u, D),
                          ts.Rows(y.o2, w, D), None, s2)

    def follow():
        ts.attn_beam_select(select, *best, s3)
        for i, y in enumerate(layers):
            ts.attn_kv_reorder(y.desc(c), best[2], beams, i == 0)

    for y in layers:
        y.states.Tq = B
    parts = [attend, follow]
    if graph:
        hip = pu.Hip()
        st = hip.stream()
        ready = [hip.capture(st, f) for f in parts]
        parts = [lambda ex=ex: hip("hipGraphLaunch", ex, st) for ex in ready]
    token = np.array([told[b // beams][-1] for b in range(B)])
    score = np.where(np.arange(B) % beams == 0, 0.0, -np.inf).astype(np.float32)
    over = np.zeros(B, np.uint8)
    moved = shared = 0
    for step in range(steps):
        c.kv_len = np.array([len(h) + 1 for h in hist], np.int32)
        c.bufs["kv_len"].upload(c.kv_len)
        for b in range(B):
            hist[b].append(int(token[b]))
        for y in layers:
            for buf, x in zip(y.ins, (y.q, y.k, y.v)):
                buf.upload(x[token])
        ts.synchronize()
        parts[0]()
        ts.synchronize()
        x = np.zeros((B, Hq * D), np.float32)
        for y in layers:
            O, bound = pu.attend_ref(Tokens(y, hist), y.q[token], Hq, 1)
            o1 = y.o1.download(np.uint16).reshape(B, Hq, D)
            assert np.all(np.abs(f32(o1) - O) <= bound), step
            t = y.states
            t.q[:B] = o1.reshape(B, -1)
            o2 = f32(y.o2.download(np.uint16)).reshape(B, Hq, D)
            ref = cu.reference(t, grad=False)["o"]
            assert np.all(np.abs(o2 - ref[0][:B]) <= ref[1][:B]), step
            x += o2.reshape(B, -1)
        # Logits of the step's own: any function of what the layers gave.
        z = x @ W + (2.0 * f32(pu.normal((B, V), 900 + step)))
        z[:, eos] += 0.1 * step
        z[5, rng.integers(0, V, 50)] = -np.inf
        logits.upload(z.astype(np.float32))
        scores.upload(score)
        done.upload(over)
        ts.synchronize()
        parts[1]()
        ts.synchronize()
        got = [best[0].download(np.float32).reshape(G, beams)] + [b.download(np.int32).reshape(G, beams)
                                                                for b in best[1:]]
        test_beam.check_select(got, test_beam.select_ref(z.astype(np.float32).astype(np.float64), score, over, eos, G,
                                                         beams, beams))
        score, token, parent = (g.reshape(-1) for g in got)
        moved += int(np.sum(parent != np.arange(B)))
        assert np.all(token >= 0)
        hist = [list(hist[p]) for p in parent]
        over = (over[parent].astype(bool) | (token == eos)).astype(np.uint8)
        table = c.bufs["table"].download(np.int32).reshape(B, c.cols)
        shared += int(np.sum(table[1::beams, 0] == table[::beams, 0]))
    print("moved", moved, "shared pages", shared, "done", over.sum(), flush=True)
    assert moved > steps and shared > 0


def test_beam_selection_of_two_streams_and_replays():
    """Two selections at once with a workspace each, eager and replayed, give what they give alone."""
    hip = pu.Hip()
    shapes = [(2, 4, 60001, 8, 16), (1, 16, 30000, 40, 32)]
    calls = []
    for i, (B, beams, V, K, bits) in enumerate(shapes):
        bufs = {"x": ts.DeviceBuffer(B * beams * V * bits // 8), "s": ts.DeviceBuffer(4 * B * beams)}
        b = ts.Beams(bufs["x"], V, bits, B, beams, V, K, bufs["s"])
        bufs["w"] = ts.DeviceBuffer(ts.attn_beam_scratch_bytes(b))
        bufs.update({j: ts.DeviceBuffer(4 * B * K) for j in range(3)})
        calls.append((b, bufs))

    def run(i):
        b, bufs = calls[i]
        ts.attn_beam_select(b, bufs[0], bufs[1], bufs[2], bufs["w"])

    streams = [hip.stream(), hip.stream()]
    run(0), run(1)
    ts.synchronize()
    graphs = [hip.capture(streams[i], lambda i=i: run(i)) for i in range(2)]
    for it in range(4):
        refs = []
        for i, (B, beams, V, K, bits) in enumerate(shapes):
            x = test_beam.logits_of(B * beams, V, bits, 100 * it + 10 * i)
            scores = -np.random.default_rng(it).random(B * beams).astype(np.float32)
            refs.append(test_beam.select_ref(test_beam.as64(x), scores, None, 0, B, beams, K))
            calls[i][1]["x"].upload(x)
            calls[i][1]["s"].upload(scores)
            for j in range(3):
                calls[i][1][j].fill_bytes(0xFF)
        ts.synchronize()
        for i in range(2):
            if it % 2:
                ts.set_stream(streams[i].value)
                run(i)
                ts.set_stream(None)
            else:
                hip("hipGraphLaunch", graphs[i], streams[i])
        ts.synchronize()
        for i, (B, beams, V, K, bits) in enumerate(shapes):
            got = [calls[i][1][j].download(np.float32 if j == 0 else np.int32).reshape(B, K) for j in range(3)]
            test_beam.check_select(got, refs[i])


@pytest.mark.parametrize("bits", [16, 32])
def test_selection_of_extreme_logits(bits):
    """Zeros of either sign are equal; a few huge and tiny logits; scores that cancel."""
    B, beams, V, K = 5, 2, 5000, 40
    x = np.zeros((B * beams, V), np.float32)
    rng = np.random.default_rng(5)
    x[0:2] = np.where(rng.random((2, V)) < 0.5, -0.0, 0.0)
    x[2:4] = -1e30
    x[2, 4000:4010], x[3, 5] = 1e30, -np.inf
    x[4:6] = rng.standard_normal((2, V)) * 1e-30
    x[6:8] = rng.standard_normal((2, V)) * 3e37
    x[8:10] = -1000.0 + rng.standard_normal((2, V))
    x = f32(bf16(x))
    scores = np.array([-0.0, 0.0, 0, 0, 1, 1, -5, 5, 1e30, 1e-30], np.float32)
    ref = test_beam.select_ref(x.astype(np.float64), scores, None, 0, B, beams, K)
    test_beam.check_select(test_beam.select(bf16(x) if bits == 16 else x, scores, None, 0, B, beams, V, K), ref)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("V", [600, 40000])
def test_selection_under_masks_of_the_lowest_value(bits, V):
    """Banned tokens have the type's lowest finite value: the first ones, nearly all, all but the last."""
    B, beams, K = 2, 4, 6
    low = f32(np.array([0xFF7F], np.uint16))[0] if bits == 16 else np.finfo(np.float32).min
    x = f32(test_beam.logits_of(B * beams, V, 16, 77)).copy()
    x[0, :V // 2] = low
    x[1, 10:] = low
    x[2, :V - 1] = low
    x[3, ::2] = low
    x[4, 7:] = low
    x[5:] = low
    x[5, [3, V - 3]] = 2.0, 1.0
    scores = -np.arange(B * beams).astype(np.float32)
    ref = test_beam.select_ref(x.astype(np.float64), scores, None, 0, B, beams, K)
    test_beam.check_select(test_beam.select(bf16(x) if bits == 16 else x, scores, None, 0, B, beams, V, K), ref)
