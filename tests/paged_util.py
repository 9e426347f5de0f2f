"""A paged KV cache on the device for the tests, and the definitions of its operators in numpy: the rotation
and the quantiser in the arithmetic that the entry points promise, attention in float64."""
import ctypes

import numpy as np

import transfer_station_amd as ts
from transfer_station_amd import _lib

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def f32(b):
    return (np.asarray(b).astype(np.uint32) << 16).view(np.float32)


def bf16(x):
    """Round to nearest even; NaN stays NaN."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def normal(shape, seed, sigma=1.0):
    return ts.synth_normal_bf16(int(np.prod(shape)), seed, 0, sigma).reshape(shape)


def quantise(b):
    """bf16 rows [..., D] -> (codes [..., D/2] bytes, scales [..., D/32] bytes)."""
    x = f32(b).astype(np.float64).reshape(*b.shape[:-1], b.shape[-1] // 32, 32)
    a = np.abs(x).max(-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(a > 0, np.ceil(np.log2(a / 7.0)), -126)
        e = np.clip(e, -126, 125)
        y = np.abs(x / np.exp2(e)[..., None])
    bad = ~np.isfinite(a)
    y = np.where(bad[..., None], 0, y)
    far = np.abs(y[..., None] - LEVELS)
    far = far - 1e-9 * (np.arange(8) % 2 == 0)  # ties to the even code
    code = far.argmin(-1) + 8 * np.signbit(x)
    code = np.where(bad[..., None], 0, code).reshape(*b.shape).astype(np.uint8)
    scale = np.where(bad, 255, np.where(bad, 0, e) + 127).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def values4(codes, scales):
    """The float64 values of 4-bit rows; NaN under scale 255."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*scales.shape, 32)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    x = LEVELS[c & 7] * (1.0 - 2.0 * (c >> 3)) * s[..., None]
    return x.reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def rotate(b, pos, rope, rot, pairs):
    """bf16 rows [n][heads][D] at positions pos, as the append entry point promises: float32 products and
    sums, one rounding."""
    if not rot:
        return b
    x, half = f32(b), rot // 2
    c, s = rope[pos][:, None, :half], rope[pos][:, None, half:]
    r = x[..., :rot]
    x1, x2 = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :half], r[..., half:])
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    y = np.stack([y1, y2], -1).reshape(r.shape) if pairs else np.concatenate([y1, y2], -1)
    return np.concatenate([bf16(y), b[..., rot:]], -1)


def rope_table(rows, rot):
    half = max(1, rot // 2)
    a = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(half) / half)
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


class Cache:
    """seqs: (new tokens, length) of each sequence. The pages lie anywhere; what no token fills is NaN."""

    def __init__(self, seqs, Hkv, D, page, bits, seed, spare=2, cols=None):
        self.seqs, self.Hkv, self.D, self.page, self.bits = seqs, Hkv, D, page, bits
        self.B = len(seqs)
        used = [-(-max(k, 0) // page) for _, k in seqs]
        self.cols = cols or max(used + [1]) + 1
        self.pages = sum(used) + spare
        order = np.random.default_rng(seed).permutation(self.pages).astype(np.int32)
        self.table = np.full((self.B, self.cols), -1, np.int32)
        at = 0
        for b, n in enumerate(used):
            m = min(n, self.cols)
            self.table[b, :m] = order[at:at + m]
            at += n
        n = [a for a, _ in seqs]
        self.start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.N = int(self.start[-1])
        self.kv_len = np.array([k for _, k in seqs], np.int32)
        rb = 2 * D if bits == 16 else D // 2
        self.k = np.full((self.pages, Hkv, page, rb), 0xFF, np.uint8)
        self.v = self.k.copy()
        self.ks = np.full((self.pages, Hkv, page, D // 32), 0xFF, np.uint8)
        self.vs = self.ks.copy()
        self.bufs = {}

    def places(self, b, lo, hi):
        j = np.arange(lo, hi)
        return self.table[b, j // self.page], j % self.page

    def put(self, b, lo, K, V):
        """bf16 rows [n][Hkv][D] as tokens lo .. of sequence b."""
        pg, at = self.places(b, lo, lo + len(K))
        for x, sc, rows in ((self.k, self.ks, K), (self.v, self.vs, V)):
            if self.bits == 4:
                x[pg, :, at], sc[pg, :, at] = quantise(rows)
            else:
                x[pg, :, at] = np.ascontiguousarray(rows).view(np.uint8).reshape(*rows.shape[:2], 2 * self.D)

    def get(self, b, lo, hi):
        """float64 rows [n][Hkv][D] of K and of V."""
        pg, at = self.places(b, lo, hi)
        out = []
        for x, sc in ((self.k, self.ks), (self.v, self.vs)):
            if self.bits == 4:
                out.append(values4(x[pg, :, at], sc[pg, :, at]))
            else:
                out.append(f32(np.ascontiguousarray(x[pg, :, at]).view(np.uint16)).astype(np.float64))
        return out

    def fill(self, seed):
        for b, (_, n) in enumerate(self.seqs):
            n = min(max(n, 0), self.cols * self.page)
            if n:
                self.put(b, 0, normal((n, self.Hkv, self.D), seed + 2 * b),
                         normal((n, self.Hkv, self.D), seed + 2 * b + 1))

    def device(self):
        for name in ("k", "v", "ks", "vs", "table", "kv_len", "start"):
            arr = getattr(self, name)
            if name in self.bufs:
                self.bufs[name].upload(arr)
            else:
                self.bufs[name] = ts.DeviceBuffer.from_array(arr)
        d = self.bufs
        return ts.KvCache(d["k"], d["v"], d["table"], d["kv_len"], d["start"], self.B, self.cols, self.pages,
                          self.page, self.Hkv, self.D, self.bits, d["ks"] if self.bits == 4 else None,
                          d["vs"] if self.bits == 4 else None)

    def download(self):
        for name in ("k", "v", "ks", "vs"):
            arr = getattr(self, name)
            setattr(self, name, self.bufs[name].download(np.uint8).reshape(arr.shape))


def attend_ref(cache, q, Hq, causal, scale=0.0, softcap=0.0, slopes=None, hidden=()):
    """(O, bound) in float64 for bf16 q [N][Hq][D]. hidden: (sequence, page column) whose keys are none.

    bound: how far a right kernel may be off. With w the softmax weights and A = sum w |v|, an output is
    sum w v; P enters the product rounded to bf16 (2^-8 of each weight), the result is rounded to bf16
    (2^-8 of it); a score that is off by d moves every weight by a factor of e^(2d) at most, where d counts
    the dot product's D + 8 roundings in fp32 and eight of the score itself (its products, the cap's tanh,
    the distance), 2^-24 each; exp2 is good to 2^-21 and enters once per rescale (a tile of 32 keys) and once
    per weight; sums over the keys add a rounding of 2^-24 per key."""
    D, g = cache.D, Hq // cache.Hkv
    scale = scale or D ** -0.5
    O, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b, (n, kv) in enumerate(cache.seqs):
        kend = min(max(kv, 0), cache.cols * cache.page)
        if not n:
            continue
        r0 = cache.start[b]
        pos = kv - n + np.arange(n)
        if not kend:
            continue
        K, V = cache.get(b, 0, kend)
        j = np.arange(kend)
        show = np.ones((n, kend), bool) if not causal else j[None, :] <= pos[:, None]
        for hb, col in hidden:
            if hb == b:
                show &= (j // cache.page != col)[None, :]
        for h in range(Hq):
            x, k = f32(q[r0:r0 + n, h]).astype(np.float64), K[:, h // g]
            v = np.where(show.any(0)[:, None], V[:, h // g], 0.0)
            with np.errstate(invalid="ignore"):
                t = scale * (x @ k.T)
                mag = scale * (np.abs(x) @ np.abs(k).T)
                if softcap:
                    t = softcap * np.tanh(t / softcap)
                    mag = mag + softcap
                if slopes is not None:
                    d = float(slopes[h]) * np.abs(pos[:, None] - j)
                    t = t - d
                    mag = mag + np.abs(d)
                t = np.where(show, t, -np.inf)
                mag = np.where(show, mag, 0.0)
                w = np.exp(t - np.where(show.any(1), t.max(1), 0.0)[:, None])
            w = w / np.maximum(w.sum(1, keepdims=True), 1e-300)
            o, A = w @ v, w @ np.abs(v)
            delta = 2 * ((D + 16) * 2.0 ** -24 * mag.max(1) + 2.0 ** -21 * (kend / 32 + 2))
            bound[r0:r0 + n, h] = 2.0 ** -8 * np.abs(o) + A * (2.0 ** -8 * 1.01 + delta[:, None] +
                                                               kend * 2.0 ** -24) + 1e-30
            O[r0:r0 + n, h] = o
    return O, bound


def attend(cache, q, Hq, causal, scale=0.0, softcap=0.0, slopes=None, max_q=None, max_kv=None, pad=3,
           stride=0, desc=None, poison=0xFF):
    """O [N][Hq][D] as float32, from q in a wider buffer between guards; rows behind the last sequence and
    between rows have to stay as they were (bytes `poison`)."""
    N, D = cache.N, cache.D
    T = N + pad
    tok = Hq * D + stride
    qh = np.full((T, tok), 0xFFFF, np.uint16)
    qh[:N, :Hq * D] = q.reshape(N, -1)
    desc = desc or cache.device()
    sc = ts.Scores(scale, softcap, None)
    with ts.DeviceBuffer.from_array(qh) as dq, ts.DeviceBuffer(T * tok * 2) as do, \
            ts.DeviceBuffer(ts.attn_flash_scratch_bytes(D, 128)) as ds, \
            ts.DeviceBuffer.from_array(np.asarray(slopes if slopes is not None else [0], np.float32)) as dl:
        do.fill_bytes(poison)
        ds.fill_bytes(0xFF)
        if slopes is not None:
            sc.slopes = dl.ptr
        ts.attn_paged(desc, ts.Rows(dq, tok, D), ts.Rows(do, tok, D), T, Hq, causal, sc,
                      max_q or max([n for n, _ in cache.seqs] + [1]),
                      max_kv or max([k for _, k in cache.seqs] + [1]), ds)
        ts.synchronize()
        raw = do.download(np.uint16).reshape(T, tok)
    assert np.all(raw[N:] == poison * 0x101) and np.all(raw[:, Hq * D:] == poison * 0x101)
    return f32(raw[:N, :Hq * D]).reshape(N, Hq, D)


def memcpy_to(ptr, arr):
    arr = np.ascontiguousarray(arr)
    _lib.check(_lib.lib().attn_dev_memcpy_htod(ctypes.c_void_p(ptr), arr.ctypes.data, arr.nbytes), "hipMemcpy")


class Hip:
    """The few calls of the HIP runtime that the tests make beside the library, which links it: streams and
    graphs."""

    def __init__(self):
        _lib.lib()
        self.h = ctypes.CDLL("libamdhip64.so.7")

    def __call__(self, name, *args):
        _lib.check(getattr(self.h, name)(*args), name)

    def stream(self):
        s = ctypes.c_void_p()
        self("hipStreamCreate", ctypes.byref(s))
        return s

    def capture(self, stream, f):
        """f's launches on the stream as an executable graph."""
        graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
        ts.set_stream(stream.value)
        try:
            self("hipStreamBeginCapture", stream, 2)  # relaxed
            f()
            self("hipStreamEndCapture", stream, ctypes.byref(graph))
        finally:
            ts.set_stream(None)
        self("hipGraphInstantiate", ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0))
        return ex
