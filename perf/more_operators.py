"""The operators of an encoder-decoder model as its training and its beam search use them: cross attention of
decoder tokens to an encoder's states of another length, its gradients, the choice of the beams that go on, and
the paged cache's sequences following their parents.

A case's "op" is
  "cross"    attention of each sequence's rows over its own encoder states, with the log-sum-exp of each row.
             K and V are the heads of one projection of the encoder's states. Lengths follow from the case alone:
             q rows (k states) at most, fewer by up to the share q_spread (k_spread); `empty` sequences have no
             states. Packed batches name their rows by starts; in padded ones every sequence has the same room,
             and what lies behind its length is anything. `pad` rows stand behind the last sequence's.
  "step"     the same, and the gradients of q, k and v: what a training step makes of a layer.
  "select"   the K best continuations of each batch entry's beams over the vocabulary: score + log-softmax.
  "reorder"  sequences of the paged cache continue their parents: full pages are shared through the table, the
             tokens of the last page are copied. In 4 bits those tokens are read back, as the values that they
             stand for.
"""
import math
import random

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _cross(op, B, q, k, Hq, Hkv, D, name=None, **more):
    c = {"op": op, "B": B, "q": q, "k": k, "Hq": Hq, "Hkv": Hkv, "D": D, "q_spread": 0.0, "k_spread": 0.0,
         "empty": 0, "padded": 0, "pad": 0}
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def _select(B, beams, V, K, bits, name=None, **more):
    c = {"op": "select", "B": B, "beams": beams, "V": V, "K": K, "bits": bits, "done": 0, "banned": 0}
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def _reorder(groups, beams, kv, prompt, Hkv, D, page, bits, name=None, spread=0.0):
    c = {"op": "reorder", "groups": groups, "beams": beams, "kv": kv, "prompt": prompt, "Hkv": Hkv, "D": D,
         "page": page, "bits": bits, "spread": spread}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # One decoder token over one encoder's states: the smallest call, made once per layer and token.
        _cross("cross", 1, 1, 1500, 16, 16, 64, name="cross_b1"),
        # Five beams each of 16 inputs: the beams of an input share its states.
        _cross("cross", 16, 5, 1500, 16, 16, 64, k_spread=0.5, name="cross_beams"),
        # A serving batch of single tokens over long documents' states.
        _cross("cross", 64, 1, 8192, 32, 8, 128, k_spread=0.6, padded=1, name="cross_b64_8k"),
        # Decoder prompts of any lengths over the states of 8 documents.
        _cross("cross", 8, 700, 4001, 32, 8, 128, q_spread=0.7, k_spread=0.5, pad=19, name="cross_prompts"),
        # A training step on a few short sentences.
        _cross("step", 3, 37, 50, 8, 8, 64, q_spread=0.4, k_spread=0.4, name="step_short"),
        # Image tokens that attend to a text of 77 tokens: many rows, few states.
        _cross("step", 4, 4096, 77, 10, 10, 64, name="step_image"),
        # A training step of an ordinary ragged batch, padded, one input without states.
        _cross("step", 8, 1000, 1500, 16, 16, 80, q_spread=0.6, k_spread=0.6, padded=1, empty=1,
               name="step_ragged"),
        # The largest: grouped heads at the sizes of the 4k prefill.
        _cross("step", 2, 4096, 4096, 32, 8, 128, name="step_4k"),
        # The beams of one input, a vocabulary that is no multiple of anything.
        _select(1, 4, 50257, 8, 32, done=1, name="select_b1"),
        # A serving batch's beams over a large vocabulary.
        _select(64, 8, 128256, 16, 16, banned=300, name="select_b64"),
        # The beams of one input share its prompt and differ in what they generated.
        _reorder(1, 4, 777, 700, 8, 128, 16, 16, name="reorder_b1"),
        # A serving batch's beams in the 4-bit cache.
        _reorder(48, 5, 1000, 800, 8, 128, 64, 4, spread=0.1, name="reorder4_b48"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more call of the same kinds."""
    while True:
        op = rng.choice(["cross", "cross", "cross", "step", "step", "step", "select", "select", "reorder"])
        Hkv = rng.choice([1, 2, 4, 8, 8, 16])
        D = rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256])
        if op == "select":
            beams = rng.randint(1, 16)
            c = _select(_log_int(rng, 1, 96), beams, _log_int(rng, 1000, 260000),
                        max(1, beams * rng.choice([1, 1, 2]) - rng.choice([0, 0, 1])), rng.choice([16, 32]),
                        done=rng.choice([0, 1]), banned=rng.choice([0, 0, rng.randint(1, 500)]))
            if c["B"] * beams * c["V"] <= 6e7:
                return c
            continue
        if op == "reorder":
            bits = rng.choice([16, 4])
            prompt = _log_int(rng, 1, 2000)
            c = _reorder(_log_int(rng, 1, 64), rng.randint(2, 12), prompt + _log_int(rng, 1, 300), prompt, Hkv,
                         rng.choice([64, 128, 256]) if bits == 4 else D, rng.choice([16, 32, 64, 128]), bits,
                         spread=rng.choice([0.0, 0.4]))
            if c["groups"] * c["beams"] * (c["kv"] - prompt + 2 * c["page"]) * Hkv * c["D"] <= 4e8 and \
                    c["groups"] * c["kv"] * Hkv * c["D"] <= 2e8:
                return c
            continue
        g = rng.choice([1, 1, 2, 4, 8])
        kind = rng.choice(["token", "rows", "many"])
        B = _log_int(rng, 1, 64) if kind == "token" else _log_int(rng, 1, 12)
        q = rng.randint(1, 8) if kind == "token" else _log_int(rng, 8, 200) if kind == "rows" else \
            _log_int(rng, 200, 4096)
        # Through a single state nothing flows back to q and k but roundings: steps have two and more.
        c = _cross(op, B, q, _log_int(rng, 1 if op == "cross" else 2, 16384), g * Hkv, Hkv, D,
                   q_spread=rng.choice([0.0, 0.5, 0.9]), k_spread=rng.choice([0.0, 0.5, 0.95]),
                   empty=rng.choice([0, 0, 1]) if B > 1 else 0, padded=rng.choice([0, 1]), pad=rng.choice([0, 0, rng.randint(1, 40)]))
        w = work(c)
        if w["flops"] <= (2e11 if op == "cross" else 6e11) and w["bytes"] <= 6e8 and \
                B * c["Hq"] * q * c["k"] <= 5e8 and B * c["k"] * c["Hq"] * D <= 3e8:
            return c


def _lengths(c):
    """(rows, states) of each sequence of a cross attention."""
    rng = random.Random(11 + c["B"] + c["k"])
    n, m = [], []
    for b in range(c["B"]):
        n.append(c["q"] if b == 0 else max(1, round(c["q"] * (1 - c["q_spread"] * rng.random()))))
        m.append(c["k"] if b == 0 else max(1, round(c["k"] * (1 - c["k_spread"] * rng.random()))))
    for b in range(c["empty"]):
        m[c["B"] - 1 - b] = 0
    return n, m


def _tokens(c):
    """Tokens of each sequence of a reordered cache: those of a group have the same number."""
    rng = random.Random(5 + c["groups"] + c["kv"])
    out = []
    for g in range(c["groups"]):
        n = c["kv"] if g == 0 else c["kv"] - int((c["kv"] - c["prompt"]) * c["spread"] * rng.random())
        out += [n] * c["beams"]
    return out


def _parents(c):
    """Parent of each sequence: beams that go on keep their place, the places of the others are taken by theirs."""
    rng = random.Random(17 + c["groups"] + c["beams"])
    out = []
    for g in range(c["groups"]):
        stays = [i for i in range(c["beams"]) if rng.random() < 0.5] or [rng.randrange(c["beams"])]
        out += [g * c["beams"] + (i if i in stays else rng.choice(stays)) for i in range(c["beams"])]
    return out


def work(c):
    if c["op"] == "select":
        rows = c["B"] * c["beams"]
        return {"bytes": rows * (c["V"] * c["bits"] // 8 + 4) + 12 * c["B"] * c["K"], "flops": 4 * rows * c["V"]}
    if c["op"] == "reorder":
        n, parent, page = _tokens(c), _parents(c), c["page"]
        row = 2 * c["Hkv"] * (2 * c["D"] if c["bits"] == 16 else c["D"] // 2 + c["D"] // 32)
        moved = [i for i, p in enumerate(parent) if p != i]
        src = {parent[i] for i in moved}
        total = sum(n[i] % page for i in moved) * row + sum(n[i] % page for i in src) * row
        total += 4 * sum(n[i] // page for i in moved) + 4 * sum(n[i] // page for i in src) + 4 * len(n)
        if c["bits"] == 4:
            total += sum(t % page for t in n) * (row + 2 * c["Hkv"] * 2 * c["D"])
        return {"bytes": total, "flops": 0}
    n, m = _lengths(c)
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    q, k, pairs = 2 * sum(n) * Hq * D, 2 * sum(m) * Hkv * D, sum(x * y for x, y in zip(n, m))
    lse = 4 * sum(n) * Hq
    if c["op"] == "cross":
        return {"bytes": 2 * q + 2 * k + lse, "flops": 4 * D * Hq * pairs}
    return {"bytes": 4 * q + 4 * k + lse, "flops": 14 * D * Hq * pairs}


# ---- states ----------------------------------------------------------------------------------
def _starts(lengths, room):
    """Each sequence's first row, and all sequences' rows: packed, or with the same room for each."""
    at, out = 0, []
    for n in lengths:
        out.append(at)
        at += room if room else n
    return out + [at], at


def prepare(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").bfloat16()

    def tensor(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    if c["op"] == "select":
        B, beams, V = c["B"], c["beams"], c["V"]
        rows = B * beams
        x = 2.5 * torch.randn(rows, V, generator=gen, device="cuda")
        if c["banned"]:
            x[:, torch.randint(0, V, (c["banned"],), generator=gen, device="cuda")] = -math.inf
        scores = -8.0 * torch.rand(B, beams, generator=gen, device="cuda")
        s = {"case": c, "logits": x if c["bits"] == 32 else x.bfloat16(),
             "scores": scores.sort(descending=True).values.reshape(rows).contiguous(), "done_token": 2,
             "done": (torch.rand(rows, generator=gen, device="cuda") < 0.2).to(torch.uint8) if c["done"] else None}
        s["score"] = torch.zeros(B, c["K"], dtype=torch.float32, device="cuda")
        s["token"] = torch.zeros(B, c["K"], dtype=torch.int32, device="cuda")
        s["parent"] = torch.zeros(B, c["K"], dtype=torch.int32, device="cuda")
        return s

    if c["op"] == "reorder":
        G, beams, page, Hkv, D = c["groups"], c["beams"], c["page"], c["Hkv"], c["D"]
        B, kv = G * beams, _tokens(c)
        shared = c["prompt"] // page
        cols = -(-c["kv"] // page) + 1
        pages = G * shared + B * (cols - shared)
        # The pages of the prompt belong to a group, those behind it to a sequence; they lie anywhere.
        order = torch.randperm(pages, generator=gen, device="cuda").int()
        j = torch.arange(cols, device="cuda")[None, :]
        b = torch.arange(B, device="cuda")[:, None]
        at = torch.where(j < shared, b // beams * shared + j, G * shared + b * (cols - shared) + j - shared)
        rem = [n % page for n in kv]
        start = [0]
        for r in rem:
            start.append(start[-1] + r)
        s = {"case": c, "pages": pages, "cols": cols, "table": order[at].contiguous(), "kv_len": tensor(kv),
             "parent": tensor(_parents(c)), "q_start": tensor(start), "T": max(1, start[-1])}
        for x in ("k", "v"):
            if c["bits"] == 4:
                s[x] = torch.randint(0, 256, (pages, Hkv, page, D // 2), generator=gen, device="cuda",
                                     dtype=torch.uint8)
                s[x + "_scale"] = torch.randint(118, 132, (pages, Hkv, page, D // 32), generator=gen,
                                                device="cuda", dtype=torch.uint8)
                s[x + "_out"] = torch.zeros(s["T"], Hkv, D, dtype=torch.bfloat16, device="cuda")
            else:
                s[x] = normal(pages, Hkv, page, D)
        return s

    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    n, m = _lengths(c)
    qs, Tq = _starts(n, c["q"] if c["padded"] else 0)
    ks, Tk = _starts(m, c["k"] if c["padded"] else 0)
    Tq, Tk = Tq + c["pad"], max(1, Tk + c["pad"])
    s = {"case": c, "Tq": Tq, "Tk": Tk, "q_start": tensor(qs), "k_start": tensor(ks), "q_len": tensor(n),
         "k_len": tensor(m)}
    s["q"] = normal(Tq, Hq, D)
    s["kv"] = normal(Tk, 2 * Hkv, D)
    s["o"] = torch.zeros(Tq, Hq, D, dtype=torch.bfloat16, device="cuda")
    s["lse"] = torch.zeros(Tq, Hq, dtype=torch.float32, device="cuda")
    if c["op"] == "step":
        s["do"] = normal(Tq, Hq, D)
        s["dq"] = torch.zeros(Tq, Hq, D, dtype=torch.bfloat16, device="cuda")
        s["dkv"] = torch.zeros(Tk, 2 * Hkv, D, dtype=torch.bfloat16, device="cuda")
    return s


# ---- the framework's operators ---------------------------------------------------------------
def _handles(s):
    """What a program makes once and keeps: descriptions of its tensors and calls, and workspaces."""
    import transfer_station_amd as ts
    c = s["case"]

    def rows(x):
        return ts.Rows(x.data_ptr(), x.stride(0), x.stride(1))

    def space(n):
        return torch.empty(n, dtype=torch.uint8, device="cuda")

    if c["op"] == "select":
        done = s["done"]
        call = ts.Beams(s["logits"].data_ptr(), s["logits"].stride(0), c["bits"], c["B"], c["beams"], c["V"],
                        c["K"], s["scores"].data_ptr(), None if done is None else done.data_ptr(),
                        s["done_token"])
        return {"ts": ts, "call": call, "scratch": space(ts.attn_beam_scratch_bytes(call))}
    if c["op"] == "reorder":
        four = c["bits"] == 4
        h = {"ts": ts,
             "cache": ts.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(),
                                 s["kv_len"].data_ptr(), s["q_start"].data_ptr(), c["groups"] * c["beams"],
                                 s["cols"], s["pages"], c["page"], c["Hkv"], c["D"], c["bits"],
                                 s["k_scale"].data_ptr() if four else None,
                                 s["v_scale"].data_ptr() if four else None)}
        if four:
            h.update(k_out=rows(s["k_out"]), v_out=rows(s["v_out"]))
        return h

    def spans(x, T, most):
        if c["padded"]:
            return ts.Spans(s[x + "_start"].data_ptr(), T, most, s[x + "_len"].data_ptr())
        return ts.Spans(s[x + "_start"].data_ptr(), T, most)

    call = ts.CrossCall(spans("q", s["Tq"], c["q"]), spans("k", s["Tk"], c["k"]), c["B"], c["Hq"], c["Hkv"],
                        c["D"])
    k, v = s["kv"].split([c["Hkv"], c["Hkv"]], 1)
    h = {"ts": ts, "call": call, "q": rows(s["q"]), "k": rows(k), "v": rows(v), "o": rows(s["o"]),
         "scratch": space(ts.attn_cross_scratch_bytes(call))}
    if c["op"] == "step":
        dk, dv = s["dkv"].split([c["Hkv"], c["Hkv"]], 1)
        h.update(do=rows(s["do"]), dq=rows(s["dq"]), dk=rows(dk), dv=rows(dv),
                 grad_scratch=space(ts.attn_cross_grad_scratch_bytes(call)))
    return h


def _run_own(s):
    c = s["case"]
    if "handles" not in s:
        s["handles"] = _handles(s)
    h = s["handles"]
    ts = h["ts"]
    if c["op"] == "select":
        ts.attn_beam_select(h["call"], s["score"].data_ptr(), s["token"].data_ptr(), s["parent"].data_ptr(),
                            h["scratch"].data_ptr())
        return {"score": s["score"], "token": s["token"], "parent": s["parent"]}
    if c["op"] == "reorder":
        ts.attn_kv_reorder(h["cache"], s["parent"].data_ptr(), c["beams"], 1)
        if c["bits"] == 16:
            return {"table": s["table"], "k": s["k"], "v": s["v"]}
        ts.attn_kv_read(h["cache"], h["k_out"], h["v_out"], s["T"], c["page"])
        return {"table": s["table"], "k": s["k_out"], "v": s["v_out"]}
    ts.attn_cross(h["call"], h["q"], h["k"], h["v"], h["o"], s["lse"].data_ptr(), h["scratch"].data_ptr())
    if c["op"] == "cross":
        return {"o": s["o"], "lse": s["lse"]}
    ts.attn_cross_grad(h["call"], h["q"], h["k"], h["v"], h["o"], s["lse"].data_ptr(), h["do"], h["dq"], h["dk"],
                       h["dv"], h["grad_scratch"].data_ptr())
    return {"o": s["o"], "lse": s["lse"], "dq": s["dq"], "dkv": s["dkv"]}


# ---- their plain forms -----------------------------------------------------------------------
def _spread(x, start, length, most):
    """Rows of all sequences, padded with zeros: [B][most][heads][D] in float32, and which of them there are."""
    i = torch.arange(most, device="cuda")
    live = i[None, :] < length[:, None]
    at = (start[:-1, None] + i[None, :]).clamp(max=x.shape[0] - 1).long()
    return torch.where(live[:, :, None, None], x[at].float(), 0.0), live, at


def _cross_plain(s):
    c = s["case"]
    B, n, m, Hq, Hkv, D = c["B"], c["q"], c["k"], c["Hq"], c["Hkv"], c["D"]
    g = Hq // Hkv
    scale = 1.0 / math.sqrt(D)

    def by_head(x, heads):  # [B][rows][Hkv heads][D] -> [B][Hkv][heads rows][D]
        return x.reshape(B, -1, Hkv, heads, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)

    def by_row(x, heads):
        return x.reshape(B, Hkv, heads, -1, D).permute(0, 3, 1, 2, 4).reshape(B, -1, Hkv * heads, D)

    q, q_live, q_at = _spread(s["q"], s["q_start"], s["q_len"], n)
    kv, k_live, k_at = _spread(s["kv"], s["k_start"], s["k_len"], m)
    q, k, v = by_head(q, g), by_head(kv[:, :, :Hkv], 1), by_head(kv[:, :, Hkv:], 1)
    t = torch.matmul(q * scale, k.transpose(-1, -2).contiguous())
    t = t.masked_fill(~k_live[:, None, None, :], -math.inf)
    top = t.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)  # rows without any state
    p = torch.exp(t - top)
    total = p.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    p = p / torch.where(total == 0, 1.0, total)
    s["o"][q_at[q_live]] = by_row(torch.matmul(p, v), g)[q_live].bfloat16()
    s["lse"][q_at[q_live]] = lse.reshape(B, Hq, n).transpose(1, 2)[q_live]
    if c["op"] == "cross":
        return {"o": s["o"], "lse": s["lse"]}
    do = by_head(_spread(s["do"], s["q_start"], s["q_len"], n)[0], g)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    del dp
    s["dq"][q_at[q_live]] = by_row(scale * torch.matmul(ds, k), g)[q_live].bfloat16()
    dk = scale * torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    del ds
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
    s["dkv"][k_at[k_live]] = torch.cat([by_row(dk, 1), by_row(dv, 1)], 2)[k_live].bfloat16()
    return {"o": s["o"], "lse": s["lse"], "dq": s["dq"], "dkv": s["dkv"]}


def _select_plain(s):
    c = s["case"]
    B, beams, V, K = c["B"], c["beams"], c["V"], c["K"]
    x = s["logits"].double()  # candidates next to each other keep their order
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    x = x + s["scores"].double()[:, None]
    if s["done"] is not None:
        over = s["done"].bool()[:, None]
        x = x.masked_fill(over, -math.inf)
        x[:, s["done_token"]] = torch.where(over[:, 0], s["scores"].double(), x[:, s["done_token"]])
    x = x.reshape(B, beams * V)
    last = x.topk(K, -1).values[:, -1:]
    more, same = x > last, x == last
    keep = more | (same & (same.cumsum(-1, dtype=torch.int32) <= K - more.sum(-1, keepdim=True)))
    at = keep.nonzero()[:, 1].reshape(B, K)  # lowest index first
    best, order = x.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    none = best == -math.inf
    first = beams * torch.arange(B, device="cuda")[:, None]
    s["score"].copy_(best)
    s["token"].copy_(torch.where(none, -1, at % V))
    s["parent"].copy_(torch.where(none, first, first + at // V))
    return {"score": s["score"], "token": s["token"], "parent": s["parent"]}


def _values(codes, scales):
    """The float32 values that 4-bit rows stand for."""
    lut = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    x = torch.stack([lut[(codes & 15).int()], lut[(codes >> 4).int()]], -1)
    x = x.reshape(*scales.shape, 32)
    return (x * (scales.int() << 23).view(torch.float32)[..., None]).reshape(*codes.shape[:-1], codes.shape[-1] * 2)


def _reorder_plain(s):
    c = s["case"]
    page, parent = c["page"], s["parent"].long()
    full, rem = s["kv_len"] // page, s["kv_len"] % page
    last = s["table"].gather(1, full[:, None].long())[:, 0].long()  # each sequence's own page
    moves = torch.arange(page, device="cuda")[None, None, :, None] < rem[:, None, None, None]
    s["table"].copy_(torch.where(torch.arange(s["cols"], device="cuda")[None, :] < full[:, None],
                                 s["table"][parent], s["table"]))

    def follow(x):
        x[last] = torch.where(moves, x[last[parent]], x[last])

    follow(s["k"])
    follow(s["v"])
    if c["bits"] == 16:
        return {"table": s["table"], "k": s["k"], "v": s["v"]}
    follow(s["k_scale"])
    follow(s["v_scale"])
    live = torch.arange(page, device="cuda")[None, :] < rem[:, None]
    N = s["q_start"][-1]

    def read(x):
        rows = _values(s[x][last], s[x + "_scale"][last]).transpose(1, 2)[live]
        s[x + "_out"][:N] = rows.bfloat16()

    read("k")
    read("v")
    return {"table": s["table"], "k": s["k_out"], "v": s["v_out"]}


def run(s):
    if own:
        return _run_own(s)
    op = s["case"]["op"]
    if op == "select":
        return _select_plain(s)
    if op == "reorder":
        return _reorder_plain(s)
    return _cross_plain(s)


# ---- from the definitions, in 64 bits --------------------------------------------------------
def _exact_cross(c, s):
    n, m = _lengths(c)
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    g = Hq // Hkv
    z = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out = {"o": z(s["o"]), "lse": z(s["lse"])}
    if c["op"] == "step":
        out.update(dq=z(s["dq"]), dkv=z(s["dkv"]))
    qs, ks = s["q_start"].tolist(), s["k_start"].tolist()
    for b in range(c["B"]):
        rows, states = slice(qs[b], qs[b] + n[b]), slice(ks[b], ks[b] + m[b])
        for h in range(Hq):
            u = h // g
            if m[b] == 0:
                out["lse"][rows, h] = -math.inf
                continue
            Q, K, V = (x.double() for x in (s["q"][rows, h], s["kv"][states, u], s["kv"][states, Hkv + u]))
            S = Q @ K.t().contiguous() * D ** -0.5
            L = torch.logsumexp(S, 1)
            P = torch.softmax(S, 1)
            O = P @ V
            out["o"][rows, h], out["lse"][rows, h] = O, L
            if c["op"] == "step":
                G = s["do"][rows, h].double()
                dS = P * (G @ V.t().contiguous() - (G * O).sum(1)[:, None])
                out["dq"][rows, h] = dS @ K * D ** -0.5
                out["dkv"][states, u] += dS.t().contiguous() @ Q * D ** -0.5
                out["dkv"][states, Hkv + u] += P.t().contiguous() @ G
    return out


def _exact_reorder(c, s):
    page, beams = c["page"], c["beams"]
    n, parent, table = _tokens(c), _parents(c), s["table"].tolist()
    new = [row[:] for row in table]
    for b, p in enumerate(parent):
        new[b][:n[b] // page] = table[p][:n[b] // page]
    pools = {x: s[x].double() for x in s if x in ("k", "v")}
    if c["bits"] == 4:
        lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
        for x in ("k", "v"):
            code = torch.stack([s[x] & 15, s[x] >> 4], -1).reshape(*s[x].shape[:-1], c["D"]).long()
            pools[x] = lut[code & 7] * (1 - 2 * (code >> 3)) * \
                torch.exp2(s[x + "_scale"].double() - 127).repeat_interleave(32, -1)
    out = {"table": None}
    for x in ("k", "v"):
        old, pool = pools[x], pools[x].clone()
        rows = []
        for b, p in enumerate(parent):
            r, j = n[b] % page, n[b] // page
            if r:
                pool[table[b][j], :, :r] = old[table[p][j], :, :r]
                rows.append(pool[table[b][j], :, :r].transpose(0, 1))
        if c["bits"] == 16:
            out[x] = pool
        else:
            out[x] = torch.zeros(s["T"], c["Hkv"], c["D"], dtype=torch.float64, device="cuda")
            if rows:
                out[x][:sum(len(r) for r in rows)] = torch.cat(rows)
    return out


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "reorder":
        return _exact_reorder(c, s)
    if c["op"] != "select":
        return _exact_cross(c, s)
    score = torch.full((c["B"], c["K"]), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        best = []
        for r in range(b * c["beams"], (b + 1) * c["beams"]):
            base = s["scores"][r].double()
            if s["done"] is not None and s["done"][r]:
                best.append(base[None])
            else:
                x = s["logits"][r].double()
                best.append(base + x.sort(descending=True).values[:c["K"]] - torch.logsumexp(x, 0))
        best = torch.cat(best).sort(descending=True).values[:c["K"]]
        score[b, :len(best)] = best
    return {"score": score, "token": None, "parent": None}
