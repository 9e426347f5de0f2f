"""The paged KV cache's operators as a serving program uses them: tokens appended to the cache with
the position rotation on the way, rows read back, and attention over the cache, for a cache held in
bf16 and for one held in 4 bits.

The cache: pages of `page` tokens, K and V [pages][Hkv][page][D]. In 4 bits a row's elements are E2M1
codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the even element low, and each 32
of them share a scale 2^(e - 127) with a byte e. Sequence b holds kv_len[b] tokens in the pages that
its row of the table names; its n_b tokens of a call are rows q_start[b] .. q_start[b + 1] - 1 of the
token tensors and the last n_b of its kv_len[b].

A case's "op" is "append" (rotate q and k, write k and v; in 4 bits the new rows are read back, as the
values that they stand for), "read" (rows of the cache to bf16) or "attend". Its lengths follow from
the case alone: kv tokens at most, fewer by up to the share kv_spread, q of them new, fewer by up to
q_spread. `pad` rows stand behind the last sequence's.
"""
import math
import random

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(op, bits, B, q, kv, Hq, Hkv, D, page, name=None, **more):
    c = {"op": op, "bits": bits, "B": B, "q": q, "kv": kv, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
         "q_spread": 0.0, "kv_spread": 0.0, "pad": 0, "rot": D if op == "append" else 0, "pairs": 0,
         "causal": 1, "softcap": 0.0, "slopes": 0}
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # One sequence's next token: the smallest call, made once per layer and token.
        _case("append", 16, 1, 1, 777, 32, 8, 128, 16, name="append_b1"),
        # Prompts of four requests, of any lengths, in a padded batch of tokens.
        _case("append", 16, 4, 4096, 4096, 32, 8, 128, 64, q_spread=0.6, kv_spread=0.6, pad=37,
              name="append_prompts"),
        # A full decode batch into the 4-bit cache; half of the head is rotated, in adjacent pairs.
        _case("append", 4, 64, 1, 500, 32, 8, 128, 32, kv_spread=0.9, rot=64, pairs=1,
              name="append4_b64"),
        # Prompt chunks of 8 requests into the 4-bit cache.
        _case("append", 4, 8, 1000, 3000, 16, 8, 128, 64, q_spread=0.5, name="append4_chunks"),
        # A long 4-bit sequence brought back as the dense K and V that attn_flash takes.
        _case("read", 4, 1, 32768, 32768, 8, 8, 128, 128, name="read4_32k"),
        # One sequence early in its generation.
        _case("attend", 16, 1, 1, 777, 32, 8, 128, 16, name="paged_b1_777"),
        # A full decode batch of sequences of all lengths.
        _case("attend", 16, 64, 1, 8192, 32, 8, 128, 64, kv_spread=0.97, name="paged_b64"),
        # Eight draft tokens of 16 sequences checked in one call, with a bias on distance.
        _case("attend", 16, 16, 8, 4001, 64, 8, 128, 32, kv_spread=0.5, slopes=1,
              name="paged_verify"),
        # A 512-token chunk of a long prompt over the 8192 keys so far.
        _case("attend", 16, 1, 512, 8192, 32, 8, 128, 64, name="paged_chunk"),
        # The full decode batch over the 4-bit cache.
        _case("attend", 4, 64, 1, 8192, 32, 8, 128, 64, kv_spread=0.5, name="paged4_b64"),
        # One sequence over a long 4-bit context, capped scores, the widest head dim.
        _case("attend", 4, 1, 1, 32768, 16, 4, 256, 128, softcap=50.0, name="paged4_b1_32k"),
        # Prompts of 6 requests over the 4-bit cache at head dim 64.
        _case("attend", 4, 6, 2000, 3000, 24, 6, 64, 16, q_spread=0.7, kv_spread=0.3, pad=9,
              name="paged4_prompts"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more call of the same kinds."""
    while True:
        bits = rng.choice([16, 4])
        kind = rng.choice(["token", "token", "draft", "prompt", "prompt"])
        op = rng.choice(["append", "attend", "attend", "attend", "read"])
        Hkv = rng.choice([1, 2, 4, 8, 8, 16])
        g = rng.choice([1, 2, 4, 4, 8, 16])
        D = rng.choice([64, 128, 128, 256] if bits == 4 else [32, 64, 80, 96, 128, 128, 192, 256])
        B = _log_int(rng, 1, 128) if kind != "prompt" else _log_int(rng, 1, 12)
        q = 1 if kind == "token" else rng.randint(2, 12) if kind == "draft" else _log_int(rng, 20, 4096)
        kv = q + rng.choice([0, _log_int(rng, 1, 16384), _log_int(rng, 16, 16384)])
        more = {"kv_spread": rng.choice([0.0, 0.3, 0.95]), "pad": rng.choice([0, 0, rng.randint(1, 40)]),
                "q_spread": rng.choice([0.0, 0.4, 0.9]) if kind == "prompt" else 0.0}
        if op == "append":
            more["rot"] = rng.choice([D, D, D // 32 * 16, 0])
            more["pairs"] = rng.choice([0, 0, 1])
        elif op == "read":
            kv = q + _log_int(rng, 1, 2000)
        else:
            more["causal"] = rng.choice([1, 1, 1, 0])
            more["softcap"] = rng.choice([0.0, 0.0, 30.0])
            more["slopes"] = rng.choice([0, 0, 1])
        c = _case(op, bits, B, q, kv, g * Hkv, Hkv, D, rng.choice([16, 32, 64, 128]), **more)
        w = work(c)
        if w["flops"] <= 1.5e11 and w["bytes"] <= 6e8 and B * g * Hkv * q * kv <= 1.5e9 and \
                B * Hkv * kv * D <= 3e8:
            return c


def _lengths(c):
    """(new tokens, tokens in the cache) of each sequence."""
    rng = random.Random(20 + c["B"] + c["kv"])
    n, kv = [], []
    for b in range(c["B"]):
        qb = c["q"] if b == 0 else max(1, round(c["q"] * (1 - c["q_spread"] * rng.random())))
        kb = c["kv"] if b == 0 else round(c["kv"] * (1 - c["kv_spread"] * rng.random()))
        n.append(qb)
        kv.append(max(kb, qb))
    return n, kv


def _positions(c):
    """How many positions the new tokens of all sequences cover, each counted once."""
    n, kv = _lengths(c)
    count, end = 0, 0
    for lo, hi in sorted((k - a, k) for a, k in zip(n, kv)):
        count += max(0, hi - max(lo, end))
        end = max(end, hi)
    return count


def work(c):
    n, kv = _lengths(c)
    row = c["Hkv"] * (2 * c["D"] if c["bits"] == 16 else c["D"] // 2 + c["D"] // 32)  # of K, or of V
    N, Hq, Hkv, D = sum(n), c["Hq"], c["Hkv"], c["D"]
    if c["op"] == "append":
        rows = N * (2 * 2 * Hq * D + 2 * 2 * Hkv * D + 2 * row) + 4 * c["rot"] * _positions(c)
        if c["bits"] == 4:
            rows += N * (2 * row + 2 * 2 * Hkv * D)  # read back
        return {"bytes": rows, "flops": 3 * N * (Hq + Hkv) * c["rot"]}
    if c["op"] == "read":
        return {"bytes": N * (2 * row + 2 * 2 * Hkv * D), "flops": 0}
    pairs = 0
    for a, k in zip(n, kv):
        pairs += a * k - (a * (a - 1) // 2 if c["causal"] else 0)
    return {"bytes": 2 * sum(kv) * row + 2 * 2 * N * Hq * D, "flops": 4 * D * Hq * pairs}


# ---- the 4-bit rows --------------------------------------------------------------------------
def _quantise(x):
    """Rows [..., D] of float32 values that bf16 holds -> (codes [..., D / 2], scales [..., D / 32]).

    The scale is the smallest power of two under which the group's largest element is at most 7, so
    that no element is further off than half the widest step; codes round to nearest, ties to the
    even code."""
    y = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    a = y.abs().amax(-1).view(torch.int32)
    e = ((a >> 23) - 2 + ((a & 0x7FFFFF) > 0x600000).int()).clamp(1, 254)
    m = (y / (e << 23).view(torch.float32)[..., None]).abs()
    code = ((m > 0.25).int() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) +
            (m > 5.0) + 8 * torch.signbit(y))
    code = code.to(torch.uint8).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), e.to(torch.uint8)


def _values(codes, scales):
    """The float32 values that 4-bit rows stand for."""
    lut = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    x = torch.stack([lut[(codes & 15).int()], lut[(codes >> 4).int()]], -1)
    x = x.reshape(*scales.shape, 32)
    s = (scales.int() << 23).view(torch.float32)
    return (x * s[..., None]).reshape(*codes.shape[:-1], codes.shape[-1] * 2)


# ---- states ----------------------------------------------------------------------------------
def _rope(c):
    """cos and sin of every position's angles, [positions][rot]: cosines first."""
    half = c["rot"] // 2
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    a = torch.arange(c["kv"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-i / max(1, half))
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    B, Hq, Hkv, D, page = c["B"], c["Hq"], c["Hkv"], c["D"], c["page"]
    n, kv = _lengths(c)
    T = sum(n) + c["pad"]
    cols = -(-c["kv"] // page) + 1
    used = [-(-k // page) for k in kv]
    pages = sum(used) + 3
    # The pages lie in the cache in the order in which they were handed out: any.
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    ends = torch.tensor(used, device="cuda").cumsum(0)
    at = torch.arange(cols, device="cuda")[None, :] + (ends - torch.tensor(used, device="cuda"))[:, None]
    table = order[at.clamp(max=pages - 1)].contiguous()
    start = [0]
    for a in n:
        start.append(start[-1] + a)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").bfloat16()

    def tensor(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    s = {"case": c, "T": T, "N": sum(n), "cols": cols, "pages": pages, "table": table,
         "kv_len": tensor(kv), "q_start": tensor(start), "max_kv": c["kv"], "max_q": c["q"]}
    for x in ("k", "v"):
        rows = normal(pages, Hkv, page, D)
        if c["bits"] == 4:
            s[x], s[x + "_scale"] = _quantise(rows.float())
        else:
            s[x] = rows
    if c["op"] == "append":
        # The projection's output: a token's query, key and value heads in one row.
        s["qkv"] = normal(T, Hq + 2 * Hkv, D)
        s["rope"] = _rope(c)
        s["q_out"] = torch.zeros(T, Hq, D, dtype=torch.bfloat16, device="cuda")
    if c["op"] == "read" or c["op"] == "append" and c["bits"] == 4:
        s["k_out"] = torch.zeros(T, Hkv, D, dtype=torch.bfloat16, device="cuda")
        s["v_out"] = torch.zeros(T, Hkv, D, dtype=torch.bfloat16, device="cuda")
    if c["op"] == "attend":
        s["q"] = normal(T, Hq, D)
        s["o"] = torch.zeros(T, Hq, D, dtype=torch.bfloat16, device="cuda")
        i = torch.arange(1, Hq + 1, device="cuda", dtype=torch.float64)
        s["slope"] = torch.exp2(-8.0 * i / Hq).float()
    return s


# ---- the framework's operators ---------------------------------------------------------------
def _handles(s):
    """What a program makes once and keeps: the cache's description, the tensors' and a workspace."""
    import transfer_station_amd as ts
    c = s["case"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]

    def rows(x):
        return ts.Rows(x.data_ptr(), x.stride(0), x.stride(1))

    four = c["bits"] == 4
    h = {"ts": ts,
         "cache": ts.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(),
                             s["kv_len"].data_ptr(), s["q_start"].data_ptr(), c["B"], s["cols"],
                             s["pages"], c["page"], Hkv, D, c["bits"],
                             s["k_scale"].data_ptr() if four else None,
                             s["v_scale"].data_ptr() if four else None)}
    if c["op"] == "append":
        q, k, v = s["qkv"].split([Hq, Hkv, Hkv], 1)
        h.update(q=rows(q), k=rows(k), v=rows(v), q_out=rows(s["q_out"]))
    if "k_out" in s:
        h.update(k_out=rows(s["k_out"]), v_out=rows(s["v_out"]))
    if c["op"] == "attend":
        h.update(q=rows(s["q"]), o=rows(s["o"]),
                 scores=ts.Scores(0.0, c["softcap"], s["slope"].data_ptr() if c["slopes"] else None),
                 scratch=torch.empty(ts.attn_flash_scratch_bytes(D, 128), dtype=torch.uint8,
                                     device="cuda"))
    return h


def _run_own(s):
    c = s["case"]
    if "handles" not in s:
        s["handles"] = _handles(s)
    h = s["handles"]
    ts = h["ts"]
    if c["op"] == "attend":
        ts.attn_paged(h["cache"], h["q"], h["o"], s["T"], c["Hq"], c["causal"], h["scores"], s["max_q"],
                      s["max_kv"], h["scratch"].data_ptr())
        return {"o": s["o"]}
    out = {}
    if c["op"] == "append":
        ts.attn_kv_append(h["cache"], h["q"], h["q_out"], h["k"], h["v"], s["T"], c["Hq"],
                          s["rope"].data_ptr(), s["rope"].shape[0], c["rot"], c["pairs"], s["max_q"])
        out["q"] = s["q_out"]
        if c["bits"] == 16:
            return {"q": s["q_out"], "k_cache": s["k"], "v_cache": s["v"]}
    ts.attn_kv_read(h["cache"], h["k_out"], h["v_out"], s["T"], s["max_q"])
    return {**out, "k": s["k_out"], "v": s["v_out"]}


# ---- their plain forms -----------------------------------------------------------------------
def _places(s):
    """Each token's position in its sequence, page and place in the page."""
    N, page = s["N"], s["case"]["page"]
    t = torch.arange(N, device="cuda")
    b = (t[:, None] >= s["q_start"][None, 1:]).sum(1)
    pos = s["kv_len"][b] - s["q_start"][b + 1] + t
    return pos, s["table"][b, pos // page], pos % page


def _rotate(x, rope, rot, pairs):
    """x [N][heads][D] in float32, each row by its row of cosines and sines."""
    half = rot // 2
    if not half:
        return x
    c, s = rope[:, None, :half], rope[:, None, half:]
    r = x[..., :rot]
    x1, x2 = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :half], r[..., half:])
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    y = torch.stack([y1, y2], -1).reshape(r.shape) if pairs else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _append(s):
    c, N = s["case"], s["N"]
    pos, pg, at = _places(s)
    q, k, v = s["qkv"][:N].float().split([c["Hq"], c["Hkv"], c["Hkv"]], 1)
    rope = s["rope"][pos]
    s["q_out"][:N] = _rotate(q, rope, c["rot"], c["pairs"]).bfloat16()
    k = _rotate(k, rope, c["rot"], c["pairs"]).bfloat16()
    for x, rows in (("k", k), ("v", v.bfloat16())):
        if c["bits"] == 4:
            codes, scales = _quantise(rows.float())
            s[x][pg, :, at] = codes
            s[x + "_scale"][pg, :, at] = scales
        else:
            s[x][pg, :, at] = rows


def _read(s):
    N = s["N"]
    pos, pg, at = _places(s)
    for x in ("k", "v"):
        if s["case"]["bits"] == 4:
            rows = _values(s[x][pg, :, at], s[x + "_scale"][pg, :, at])
        else:
            rows = s[x][pg, :, at]
        s[x + "_out"][:N] = rows.bfloat16()


def _all_rows(s, x):
    """K or V of every sequence, padded: [B][Hkv][keys][D] in float32."""
    c = s["case"]
    rows = s[x][s["table"]]
    rows = _values(rows, s[x + "_scale"][s["table"]]) if c["bits"] == 4 else rows.float()
    rows = rows.permute(0, 2, 1, 3, 4).reshape(c["B"], c["Hkv"], s["cols"] * c["page"], c["D"])
    return rows[:, :, :c["kv"]]


def _attend(s):
    c = s["case"]
    B, q, kv, Hq, Hkv, D = c["B"], c["q"], c["kv"], c["Hq"], c["Hkv"], c["D"]
    g = Hq // Hkv
    n = s["q_start"][1:] - s["q_start"][:-1]
    i = torch.arange(q, device="cuda")
    row = (s["q_start"][:-1, None] + torch.minimum(i[None, :], n[:, None] - 1)).long()  # [B][q]
    pos = (s["kv_len"] - n)[:, None] + i[None, :]
    x = s["q"][row].float() / math.sqrt(D)  # [B][q][Hq][D]
    x = x.reshape(B, q, Hkv, g, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * q, D)
    t = torch.matmul(x, _all_rows(s, "k").transpose(-1, -2).contiguous())
    t = t.reshape(B, Hkv, g, q, kv)
    if c["softcap"]:
        t = c["softcap"] * torch.tanh(t / c["softcap"])
    j = torch.arange(kv, device="cuda")
    if c["slopes"]:
        far = (pos[:, :, None] - j).abs().float()
        t = t - s["slope"].reshape(1, Hkv, g, 1, 1) * far[:, None, None]
    hide = (j[None, :] >= s["kv_len"][:, None])[:, None, :].expand(B, q, kv)
    if c["causal"]:
        hide = hide | (j > pos[:, :, None])
    t = t.masked_fill(hide[:, None, None], -math.inf)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    # Keys behind a sequence's last are another's, or nobody's.
    v = _all_rows(s, "v").masked_fill((j[None, :] >= s["kv_len"][:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.reshape(B, Hkv, g * q, kv), v)
    o = o.reshape(B, Hkv, g, q, D).permute(0, 3, 1, 2, 4).reshape(B * q, Hq, D).bfloat16()
    # A row that stands for no token repeats its sequence's last one, which follows it.
    at = torch.arange(s["N"], device="cuda")
    b = (at[:, None] >= s["q_start"][None, 1:]).sum(1)
    s["o"][:s["N"]] = o[b * q + at - s["q_start"][b]]


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "attend":
        _attend(s)
        return {"o": s["o"]}
    out = {}
    if c["op"] == "append":
        _append(s)
        out["q"] = s["q_out"]
        if c["bits"] == 16:
            return {"q": s["q_out"], "k_cache": s["k"], "v_cache": s["v"]}
    _read(s)
    return {**out, "k": s["k_out"], "v": s["v_out"]}


# ---- from the definitions, in 64 bits --------------------------------------------------------
def _exact_row4(codes, scales):
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    out = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device="cuda")
    for odd in (0, 1):
        nib = (codes.long() >> (4 * odd)) & 15
        out[..., odd::2] = lut[nib & 7] * (1 - 2 * (nib >> 3))
    return out * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _exact_quantised(x):
    """The values that rows of float64 stand for once held in 4 bits: the scale is a power of two, each
    element becomes the nearest level under it."""
    x = x.bfloat16().double()
    y = x.reshape(*x.shape[:-1], -1, 32)
    a = y.abs().amax(-1, keepdim=True)
    u = torch.exp2(torch.ceil(torch.log2(a / 7.0))).clamp_min(2.0 ** -126)
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    z = (y / u).abs()
    best, far = torch.zeros_like(z), torch.full_like(z, math.inf)
    for i in (0, 2, 4, 6, 1, 3, 5, 7):  # even codes first: they keep ties
        d = (z - lut[i]).abs()
        best = torch.where(d < far, lut[i], best)
        far = torch.minimum(d, far)
    return (best * torch.sign(y) * u).reshape(x.shape)


def _exact_rotated(x, rope, c):
    half = c["rot"] // 2
    y = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + half)
        cs, sn = rope[:, i, None], rope[:, half + i, None]
        y[..., a] = x[..., a] * cs - x[..., b] * sn
        y[..., b] = x[..., a] * sn + x[..., b] * cs
    return y


def exact(c, seed):
    s = prepare(c, seed)
    n, kv = _lengths(c)
    page, Hq, Hkv, D = c["page"], c["Hq"], c["Hkv"], c["D"]
    g = Hq // Hkv
    four = c["bits"] == 4

    def held(x, b, lo, hi):
        """Rows lo .. hi - 1 of sequence b, [hi - lo][Hkv][D]."""
        j = torch.arange(lo, hi, device="cuda")
        pg = s["table"][b].long()[j // page]
        if four:
            return _exact_row4(s[x][pg, :, j % page], s[x + "_scale"][pg, :, j % page])
        return s[x][pg, :, j % page].double()

    zeros = lambda heads: torch.zeros(s["T"], heads, D, dtype=torch.float64, device="cuda")  # noqa: E731
    at = 0
    if c["op"] == "read":
        out = {"k": zeros(Hkv), "v": zeros(Hkv)}
        for b in range(c["B"]):
            for x in ("k", "v"):
                out[x][at:at + n[b]] = held(x, b, kv[b] - n[b], kv[b])
            at += n[b]
        return out
    if c["op"] == "append":
        out = {"q": zeros(Hq)}
        if four:
            out.update(k=zeros(Hkv), v=zeros(Hkv))
        else:
            out.update(k_cache=s["k"].double(), v_cache=s["v"].double())
        for b in range(c["B"]):
            x = s["qkv"][at:at + n[b]].double()
            rope = s["rope"][kv[b] - n[b]:kv[b]].double()
            out["q"][at:at + n[b]] = _exact_rotated(x[:, :Hq], rope, c)
            k, v = _exact_rotated(x[:, Hq:Hq + Hkv], rope, c), x[:, Hq + Hkv:]
            if four:
                out["k"][at:at + n[b]], out["v"][at:at + n[b]] = _exact_quantised(k), _exact_quantised(v)
            else:
                j = torch.arange(kv[b] - n[b], kv[b], device="cuda")
                pg = s["table"][b].long()[j // page]
                out["k_cache"][pg, :, j % page], out["v_cache"][pg, :, j % page] = k, v
            at += n[b]
        return out
    o = zeros(Hq)
    for b in range(c["B"]):
        K, V = held("k", b, 0, kv[b]), held("v", b, 0, kv[b])
        j = torch.arange(kv[b], device="cuda")
        step = max(1, (1 << 25) // (kv[b] * Hq))
        for r in range(0, n[b], step):
            m = min(step, n[b] - r)
            p = kv[b] - n[b] + r + torch.arange(m, device="cuda")
            for u in range(Hkv):
                x = s["q"][at + r:at + r + m, u * g:(u + 1) * g].double()  # [m][g][D]
                t = (x.reshape(m * g, D) @ K[:, u].t().contiguous()).reshape(m, g, -1) * D ** -0.5
                if c["softcap"]:
                    t = c["softcap"] * torch.tanh(t / c["softcap"])
                if c["slopes"]:
                    t -= s["slope"][u * g:(u + 1) * g].double()[None, :, None] * \
                        (p[:, None] - j).abs().double()[:, None]
                if c["causal"]:
                    t.masked_fill_((j > p[:, None])[:, None], -math.inf)
                w = torch.softmax(t, -1)
                o[at + r:at + r + m, u * g:(u + 1) * g] = \
                    (w.reshape(m * g, -1) @ V[:, u].contiguous()).reshape(m, g, D)
        at += n[b]
    return {"o": o}
