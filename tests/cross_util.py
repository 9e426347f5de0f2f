"""Cross attention on the device for the tests, and its definition with gradients in float64, with how far a right
kernel may be off."""
import numpy as np

import transfer_station_amd as ts
from paged_util import f32, normal

E = 2.0 ** -8    # half a step of bf16, relative
E32 = 2.0 ** -24  # half a step of fp32


class Batch:
    """seqs: (rows, states) of each sequence. Packed, or (room given) padded: each sequence has room[0] rows and room[1]
    states. What no sequence names is NaN. claim: how many states the call says that there are (0: as many as there are)."""

    def __init__(self, seqs, Hq, Hkv, D, seed, room=None, claim=0, pad=3, sigma_q=1.0, stride=0, offset=0):
        self.seqs, self.Hq, self.Hkv, self.D, self.room, self.claim = seqs, Hq, Hkv, D, room, claim
        self.B, self.fine = len(seqs), (False, False)
        self.spans = {}
        for x, i, heads in (("q", 0, Hq), ("k", 1, Hkv)):
            n = [s[i] for s in seqs]
            if room:
                start = offset + room[i] * np.arange(self.B + 1)
            else:
                start = offset + np.concatenate([[0], np.cumsum(n)])
            T = max(1, int(start[-1]) + pad)
            self.spans[x] = (start.astype(np.int32), np.array(n, np.int32), T)
        self.Tq, self.Tk = self.spans["q"][2], self.spans["k"][2]
        self.live_q, self.live_k = np.zeros(self.Tq, bool), np.zeros(self.Tk, bool)
        for b in range(self.B):
            r, s = self.rows(b)
            self.live_q[r] = True
            self.live_k[s] = True
        # Rows of the tensors are wider than their heads by `stride`.
        self.q = self.tensor(self.live_q, Hq, seed, stride, sigma_q)
        self.k = self.tensor(self.live_k, Hkv, seed + 1, stride)
        self.v = self.tensor(self.live_k, Hkv, seed + 2, stride)
        self.go = self.tensor(self.live_q, Hq, seed + 3, stride)

    def tensor(self, live, heads, seed, stride, sigma=1.0):
        x = np.full((len(live), heads * self.D + stride), 0xFFFF, np.uint16)
        x[live, :heads * self.D] = normal((int(live.sum()), heads * self.D), seed, sigma)
        return x

    def rows(self, b):
        out = []
        for x in ("q", "k"):
            start, n, _ = self.spans[x]
            out.append(slice(int(start[b]), int(start[b] + n[b])))
        return out

    def head(self, x, rows, h):
        return f32(x[rows, h * self.D:(h + 1) * self.D]).astype(np.float64)


def reference(t, scale=0.0, grad=True):
    """{name: (values, bound)} of o, lse, dq, dk and dv, in float64.

    With e = 2^-8: P and dS enter their products rounded to bf16 (e of each; in two parts, e^2 = 2^-16), each result is
    rounded once (2^-8 of it).
    O and dV: off by (e + d) sum P |.| + e |result|, where d is what P is off by before its rounding: a score is off by
    (D + 8) roundings of 2^-24 of sum |q||k|, as is lse, exp2 is good to 2^-21 and enters once per tile and weight.
    dS = P (dP - delta): delta is made of the rounded O (off by what O is), or, of up to 32 states, of P dP in fp32 (off by d
    of its terms); dP and delta of D products in fp32;
    so dS is off by (e + d) |dS| + P (sum |dO| off(O) + (D + 8) 2^-24 sum |dO| (|V| + |O|)), and dQ and dK by the sums
    of that, times the factors' sizes. Sums over n terms add n 2^-24 of the terms' sizes."""
    scale = scale or t.D ** -0.5
    g = t.Hq // t.Hkv
    shape = {"o": (t.Tq, t.Hq, t.D), "lse": (t.Tq, t.Hq), "dq": (t.Tq, t.Hq, t.D), "dk": (t.Tk, t.Hkv, t.D),
             "dv": (t.Tk, t.Hkv, t.D)}
    out = {x: (np.zeros(s), np.zeros(s)) for x, s in shape.items()}
    for b, (n, m) in enumerate(t.seqs):
        rows, states = t.rows(b)
        if n and not m:
            out["lse"][0][rows] = -np.inf
        if not n or not m:
            continue
        for h in range(t.Hq):
            u = h // g
            Q, K, V, G = (t.head(x, r, i) for x, r, i in
                          ((t.q, rows, h), (t.k, states, u), (t.v, states, u), (t.go, rows, h)))
            S = scale * (Q @ K.T)
            mag = scale * (np.abs(Q) @ np.abs(K).T)
            top = S.max(1, keepdims=True)
            w = np.exp(S - top)
            total = w.sum(1, keepdims=True)
            P = w / total
            O = P @ V
            ds_ = (t.D + 16) * E32 * mag.max(1, keepdims=True)  # of a score
            d = 2 * (ds_ + 2.0 ** -21 * (m / 32 + 2)) + m * E32
            o_off = (E * 1.01 + d) * (P @ np.abs(V)) + E * np.abs(O) + 1e-30
            lse = (top + np.log(total))[:, 0]
            out["o"][0][rows, h], out["o"][1][rows, h] = O, o_off
            out["lse"][0][rows, h] = lse
            out["lse"][1][rows, h] = (ds_[:, 0] + 2.0 ** -20 + m * E32 + 8 * E32 * (np.abs(lse) + np.abs(top[:, 0])))
            if not grad:
                continue
            d = d + 8 * E32 * (np.abs(lse) + np.abs(top[:, 0]))[:, None]
            dP = G @ V.T
            dS = P * (dP - (G * O).sum(1, keepdims=True))
            Ga = np.abs(G)
            if m <= 32:
                delta_off = (P * ((d + m * E32) * np.abs(dP) + (t.D + 8) * E32 * (Ga @ np.abs(V).T))).sum(1, keepdims=True)
            else:
                delta_off = (Ga * o_off).sum(1, keepdims=True) + (t.D + 8) * E32 * (Ga * np.abs(O)).sum(1, keepdims=True)
            ds_off = d * np.abs(dS) + P * (delta_off + (t.D + 8) * E32 * (Ga @ np.abs(V).T))
            # e of P and dS in dQ, and in dK and dV
            eq, ek = (2.0 ** -16 if f else E * 1.01 for f in t.fine)
            dQ = scale * (dS @ K)
            out["dq"][0][rows, h] = dQ
            out["dq"][1][rows, h] = (scale * ((ds_off + (eq + m * E32) * np.abs(dS)) @ np.abs(K)) + E * np.abs(dQ) + 1e-30)
            n_all = n * g
            out["dk"][0][states, u] += scale * (dS.T @ Q)
            out["dk"][1][states, u] += scale * ((ds_off + (ek + n_all * E32) * np.abs(dS)).T @ np.abs(Q))
            out["dv"][0][states, u] += P.T @ G
            out["dv"][1][states, u] += ((ek + d + n_all * E32) * P).T @ Ga
        for x in ("dk", "dv"):
            out[x][1][states] += E * np.abs(out[x][0][states]) + 1e-30
    return out


def _rows(buf, tok, D):
    return ts.Rows(buf, tok, D)


def call_of(t, bufs, scale=0.0, max_q=None, max_k=None):
    def spans(x, i, most):
        start, n, T = t.spans[x]
        most = most or max([s[i] for s in t.seqs] + [1])
        if i and t.claim:
            T = most = t.claim
        bufs[x + "_start"] = ts.DeviceBuffer.from_array(start)
        if t.room:
            bufs[x + "_len"] = ts.DeviceBuffer.from_array(n)
            return ts.Spans(bufs[x + "_start"], T, most, bufs[x + "_len"])
        return ts.Spans(bufs[x + "_start"], T, most)

    call = ts.CrossCall(spans("q", 0, max_q), spans("k", 1, max_k), t.B, t.Hq, t.Hkv, t.D, scale)
    # Do dQ's kernel, and dK's and dV's, take P and dS in two parts?
    names = [p[0] for p in ts.attn_cross_plan(call, True)]
    t.fine = tuple(all(n.endswith("true>") for n in names if x in n) for x in ("_dq_", "_dkv_"))
    return call


def run(t, scale=0.0, grad=True, max_q=None, max_k=None, lse=True):
    """{name: float32 values} of what the entry points write; what no sequence names has to stay as it was."""
    bufs = {}
    call = call_of(t, bufs, scale, max_q, max_k)
    D = t.D
    for x in ("q", "k", "v", "go"):
        bufs[x] = ts.DeviceBuffer.from_array(getattr(t, x))
    r = {x: _rows(bufs[x], getattr(t, x).shape[1], D) for x in ("q", "k", "v", "go")}
    shapes = {"o": t.q.shape, "dq": t.q.shape, "dk": t.k.shape, "dv": t.v.shape}
    for x, s in shapes.items():
        bufs[x] = ts.DeviceBuffer(2 * s[0] * s[1])
        bufs[x].fill_bytes(0xFF)
        r[x] = _rows(bufs[x], s[1], D)
    bufs["lse"] = ts.DeviceBuffer(4 * t.Tq * t.Hq)
    bufs["lse"].fill_bytes(0xFF)
    guard = 4096  # bytes behind a workspace, which have to stay
    bufs["s"] = ts.DeviceBuffer(ts.attn_cross_scratch_bytes(call) + guard)
    bufs["s"].fill_bytes(0xFF)
    ts.attn_cross(call, r["q"], r["k"], r["v"], r["o"], bufs["lse"] if lse else None, bufs["s"])
    names = ["o"]
    if grad:
        bufs["gs"] = ts.DeviceBuffer(ts.attn_cross_grad_scratch_bytes(call) + guard)
        bufs["gs"].fill_bytes(0xFF)
        ts.attn_cross_grad(call, r["q"], r["k"], r["v"], r["o"], bufs["lse"], r["go"], r["dq"], r["dk"], r["dv"],
                           bufs["gs"])
        names += ["dq", "dk", "dv"]
    ts.synchronize()
    for x in ("s", "gs"):
        if x in bufs:
            assert np.all(bufs[x].download(np.uint8)[-guard:] == 0xFF), x
    out = {}
    for x in names:
        heads, live = (t.Hq, t.live_q) if x in ("o", "dq") else (t.Hkv, t.live_k)
        raw = bufs[x].download(np.uint16).reshape(shapes[x])
        assert np.all(raw[~live] == 0xFFFF) and np.all(raw[:, heads * D:] == 0xFFFF), x
        out[x] = f32(raw[:, :heads * D]).reshape(-1, heads, D)
    if lse:
        got = bufs["lse"].download(np.float32).reshape(t.Tq, t.Hq)
        assert np.all(got.view(np.uint32)[~t.live_q] == 0xFFFFFFFF)
        out["lse"] = got
    for b in bufs.values():
        b.free()
    return out


def check(t, got, ref, label=""):
    for x, y in got.items():
        live = t.live_q if x in ("o", "lse", "dq") else t.live_k
        want, bound = ref[x][0][live], ref[x][1][live]
        y = y[live].astype(np.float64)
        fine = np.isfinite(want)
        assert np.array_equal(y[~fine], want[~fine]), (label, x)
        off = np.abs(y[fine] - want[fine])
        worst = float(np.max(off / np.maximum(bound[fine], 1e-30))) if off.size else 0.0
        print("%s %-3s worst error / bound %.3f" % (label, x, worst), flush=True)
        assert np.all(off <= bound[fine]), (label, x, worst)
