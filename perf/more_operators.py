"""The operators between a decoder block's q, k, v products and its output product, as measurable cases: what one call of
each reads and answers, in plain torch (own = False) and through hipster_amd.qmm (own = True).

ops
  rope      rotary positions with several axes (time, height, width): each pair of a head's values turned by
            its axis' position times its frequency
  cache     rows of keys and values quantised to MXFP4 into the pages of their sequences, and read back as values
  attend    attention of a few new rows a sequence (decode, draft verification) over a paged MXFP4 cache
  prompt    causal attention of packed prompts of different lengths, grouped heads, bf16

A sequence has `len` keys, the last m of them from its m new rows.  A row at position p sees the keys of (p - window, p]
(window 0: all up to p).  A head's sink is a logit that takes part in the softmax and has no value.  Queries and keys are
normal with a few channels larger, as trained heads have them, so that a few keys carry most of the weight.
"""
import math

import torch

own = False

DEV = "cuda"
AXES = 3


def listed():
    return [
        # one user's decode step, text at the end of a picture: nothing but latency
        dict(name="rope_t1", op="rope", T=1, heads=40, D=128, pairs=64, style="halves", mixed=True, far=40000, dtype="f32", out="bf16"),
        # a prompt with pictures, the first quarter of each head turned
        dict(name="rope_t2000", op="rope", T=2000, heads=20, D=256, pairs=32, style="neighbours", mixed=False, far=2000, dtype="bf16", out="bf16"),
        # a decode step of 24 users: one row each
        dict(name="cache_b24", op="cache", B=24, m=1, longest=4096, Hk=8, D=128, page=64, dtype="bf16"),
        # three prompts of different lengths, whole
        dict(name="cache_b3", op="cache", B=3, m=0, longest=2048, Hk=8, D=128, page=64, dtype="bf16"),
        # one user's decode step in a short conversation
        dict(name="attend_b1", op="attend", B=1, m=1, longest=700, Hq=32, Hk=8, D=128, page=64, window=0, sinks=False, q="bf16", out="bf16"),
        # a batch of 32 users, contexts of different lengths
        dict(name="attend_b32", op="attend", B=32, m=1, longest=8192, Hq=32, Hk=8, D=128, page=64, window=0, sinks=False, q="bf16", out="bf16"),
        # one user's decode step in a long document, wide heads
        dict(name="attend_long", op="attend", B=1, m=1, longest=131072, Hq=16, Hk=4, D=256, page=256, window=0, sinks=False, q="bf16", out="bf16"),
        # five drafted rows of eight users checked at once, narrow heads with sinks, f32 in and out
        dict(name="attend_draft", op="attend", B=8, m=5, longest=3000, Hq=64, Hk=8, D=64, page=16, window=0, sinks=True, q="f32", out="f32"),
        # short prompts packed together: latency
        dict(name="prompt_b7", op="prompt", B=7, m=0, longest=300, Hq=32, Hk=8, D=128, window=0, sinks=False),
        # one prompt of ordinary length
        dict(name="prompt_2048", op="prompt", B=1, m=0, longest=2048, Hq=32, Hk=8, D=128, window=0, sinks=False),
        # a later piece of a long prompt: 512 rows behind those that are cached, wide heads
        dict(name="prompt_piece", op="prompt", B=1, m=512, longest=8000, Hq=16, Hk=2, D=256, window=0, sinks=False),
        # a long document: the largest call
        dict(name="prompt_8192", op="prompt", B=1, m=0, longest=8192, Hq=32, Hk=8, D=128, window=0, sinks=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attend", "attend", "attend", "prompt", "prompt", "prompt"])
    D = rng.choice([64, 128, 128, 256])
    Hk, g = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    if op == "rope":
        heads = rng.randint(1, 48)
        return dict(op=op, T=_spread(rng, 1, 2000 * 20 * 256 // (heads * D)), heads=heads, D=D, pairs=rng.choice([D // 2, D // 4, D // 8, rng.randint(1, D // 2)]),
                    style=rng.choice(["halves", "neighbours"]), mixed=rng.random() < 0.5, far=_spread(rng, 8, 1 << 20),
                    dtype=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16", "bf16"]))
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "cache":
        m = rng.choice([0, 1, 1, 3, 8])
        B = _spread(rng, 1, 64 if m else 8)
        longest = _spread(rng, max(8, m), 8192 if m else 3 * 2048 * 8 * 128 // (B * Hk * D))
        return dict(op=op, B=B, m=m, longest=longest, Hk=Hk, D=D, page=page, dtype=rng.choice(["f32", "bf16"]))
    window = rng.choice([0, 0, 0, 1, 128, _spread(rng, 2, 4096)])
    if op == "attend":
        m, B = rng.choice([1, 1, 1, 2, 4, 5, 8, 16]), _spread(rng, 1, 64)
        wide = rng.random() < 0.3
        return dict(op=op, B=B, m=m, longest=_spread(rng, m, max(m, min(131072, 131072 * 4 * 256 // (B * Hk * D) // (1 + m * g // 64)))), Hq=Hk * g, Hk=Hk, D=D,
                    page=page, window=window, sinks=rng.random() < 0.3, q="f32" if wide else "bf16", out="f32" if wide or rng.random() < 0.2 else "bf16")
    B, m = _spread(rng, 1, 16), rng.choice([0, 0, 0, _spread(rng, 1, 1024)])
    room = 8192 * 8192 * 32 * 128 // 2 // (B * Hk * g * D)          # visible pairs of a sequence
    held = 160_000_000 // (4 * B * Hk * D * (1 if m else 1 + g))     # tokens of a sequence whose rows take 160 MB in all
    m = min(m, 160_000_000 // (4 * B * Hk * g * D))
    longest = _spread(rng, max(1, m), max(1, m, min(16384, held, room // m if m else math.isqrt(2 * room))))
    return dict(op=op, B=B, m=m, longest=longest, Hq=Hk * g, Hk=Hk, D=D, window=window, sinks=rng.random() < 0.3)


def _lengths(c):
    """(keys, new rows) of each sequence: the first the longest, the others down to a quarter of it."""
    n = [max(1, c["longest"] - (i * 977 + (i > 0)) % max(1, c["longest"] * 3 // 4)) for i in range(c["B"])]
    return [(max(v, c["m"]), c["m"] or v) for v in n]


def _visible(length, m, window):
    """Keys that the m last rows of `length` see, in all."""
    return sum(min(p + 1, window or p + 1) for p in range(length - m, length))


# ---- inputs ----
_T = {"f32": torch.float32, "bf16": torch.bfloat16}


def _rows(g, R, heads, D, dtype):
    x = torch.randn((R, heads, D), device=DEV, generator=g)
    big = torch.randint(0, D, (max(1, D // 32),), device=DEV, generator=g)
    x[:, :, big] *= 3.0
    return x.to(_T[dtype]).view(R, heads * D)


def _pow2(e):
    """2^e for whole e in float64, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantise(x):
    """Values [..][D] -> packed codes [..][D / 2] (the even value in the low half) and scale bytes [..][D / 32]."""
    v = x.float().unflatten(-1, (-1, 32))
    amax = v.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, torch.full_like(amax, -127, dtype=torch.int32)).clamp(min=-127)
    t = (v.double() * _pow2(-e).unsqueeze(-1)).abs().float()
    code = (t > 0.25).byte()
    for border, closed in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (t >= border) if closed else (t > border)
    code = (code | (torch.signbit(v).byte() << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).byte()


def _values(q, e):
    """float32 values of packed codes [..][D / 2] with scale bytes [..][D / 32]."""
    level = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=q.device)
    v = level[torch.stack([q & 15, q >> 4], -1).flatten(-2).long()]
    return v * _pow2(e.int() - 127).float().repeat_interleave(32, -1)


def _offsets(n):
    out = [0]
    for v in n:
        out.append(out[-1] + v)
    return out


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(g, c, s, filled):
    """A paged cache [pages][Hk][page][..] with the sequences' pages in any order, its other pages free."""
    B, Hk, D, page = c["B"], c["Hk"], c["D"], c["page"]
    need = [-(-n // page) for n, _ in s["n"]]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=DEV, generator=g).int()
    table = torch.zeros((B, max(need)), dtype=torch.int32, device=DEV)
    at = _offsets(need)
    for b in range(B):
        table[b, :need[b]] = order[at[b]:at[b + 1]]
    s.update(table=table, need=need)
    for name in ("k", "v"):
        q = torch.zeros((pages, Hk, page, D // 2), dtype=torch.uint8, device=DEV)
        e = torch.zeros((pages, Hk, page, D // 32), dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 26) // (Hk * page * D))
        for i in range(0, pages if filled else 0, step):
            n = min(step, pages - i)
            q[i:i + n], e[i:i + n] = _quantise(_rows(g, n * page * Hk, 1, D, "bf16").view(n, Hk, page, D))
        s[name + "q"], s[name + "e"] = q, e


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    op, s = c["op"], dict(c=c)
    D = c["D"]
    if own:
        from hipster_amd import qmm
        s["qmm"] = qmm
    if op == "rope":
        T, P = c["T"], c["pairs"]
        freq = torch.pow(torch.tensor(1e6, dtype=torch.float64), -torch.arange(P, dtype=torch.float64) / P).float().to(DEV)
        axis = torch.arange(P) % AXES if c["mixed"] else torch.arange(P) * AXES // P
        pos = torch.randint(0, 64, (AXES, T), device=DEV, generator=g).int()           # height and width within a picture
        pos += torch.randint(max(1, c["far"] - T), c["far"] + 1, (1, 1), device=DEV, generator=g).int()
        pos[0] += torch.arange(T, device=DEV).int()
        s.update(x=_rows(g, T, c["heads"], D, c["dtype"]), freq=freq, axis=axis.byte().to(DEV), pos=pos,
                 y=torch.empty((T, c["heads"] * D), dtype=_T[c["out"]], device=DEV))
        return s
    s["n"] = _lengths(c)
    cu = _offsets([m for _, m in s["n"]])
    rows = cu[-1]
    s.update(at=cu, cu=_int(cu), lens=_int([n for n, _ in s["n"]]))
    if op == "cache":
        _cache(g, c, s, False)
        for name in ("k", "v"):
            s[name] = _rows(g, rows, c["Hk"], D, c["dtype"])
            s[name + "o"] = torch.empty((rows, c["Hk"] * D), dtype=torch.bfloat16, device=DEV)
    else:
        Hq, Hk = c["Hq"], c["Hk"]
        s["sinks"] = torch.randn(Hq, device=DEV, generator=g) if c["sinks"] else None
        s["q"] = _rows(g, rows, Hq, D, c.get("q", "bf16"))
        s["o"] = torch.empty((rows, Hq * D), dtype=_T[c.get("out", "bf16")], device=DEV)
        if op == "attend":
            _cache(g, c, s, True)
        else:
            atk = _offsets([n for n, _ in s["n"]])
            s.update(atk=atk, cuk=_int(atk), k=_rows(g, atk[-1], Hk, D, "bf16"), v=_rows(g, atk[-1], Hk, D, "bf16"))
    if own and op != "prompt":
        kv = qmm.KVMXBuf(s["kq"].shape[0], c["page"], c["Hk"], D, device=DEV)
        kv.kq, kv.ke, kv.vq, kv.ve = s["kq"], s["ke"], s["vq"], s["ve"]
        s["kv"] = kv
        if op == "attend":
            s["ws"] = torch.empty(qmm.attn_kv_ws_bytes(rows, c["Hq"], D, c["longest"]), dtype=torch.uint8, device=DEV)
    return s


# ---- one pass, plain ----
def _plain_rope(s):
    c = s["c"]
    T, H, D, P = c["T"], c["heads"], c["D"], c["pairs"]
    angle = s["pos"].double()[s["axis"].long()].t() * s["freq"].double()             # 64 bits: far positions
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    x = s["x"].float().view(T, H, D)
    y = x.clone()
    a, b = (slice(0, P), slice(P, 2 * P)) if c["style"] == "halves" else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    y[:, :, a] = x[:, :, a] * cos - x[:, :, b] * sin
    y[:, :, b] = x[:, :, b] * cos + x[:, :, a] * sin
    return {"y": y.view(T, H * D).to(_T[c["out"]])}


def _places(s):
    """Page and place in it of every row."""
    page, where = s["c"]["page"], []
    for b, (n, m) in enumerate(s["n"]):
        p = torch.arange(n - m, n, device=DEV)
        where.append((s["table"][b].long()[p // page], p % page))
    return [torch.cat(t) for t in zip(*where)]


def _plain_cache(s):
    c = s["c"]
    pg, at = _places(s)
    out = {}
    for name in ("k", "v"):
        q, e = _quantise(s[name].view(-1, c["Hk"], c["D"]))
        s[name + "q"][pg, :, at], s[name + "e"][pg, :, at] = q, e
        out[name] = _values(s[name + "q"][pg, :, at], s[name + "e"][pg, :, at]).flatten(1).bfloat16()
    return out


def _hidden(n, m, window):
    """[m][n], true where row n - m + i does not see key j."""
    p = torch.arange(n - m, n, device=DEV).unsqueeze(1)
    j = torch.arange(n, device=DEV).unsqueeze(0)
    return (j > p) | (j <= p - window) if window else j > p


def _softmax_times(score, v, hide, sink):
    """softmax over the last axis, a sink beside it, times v.  Changes score."""
    score.masked_fill_(hide, -float("inf"))
    top = score.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    return (score @ v) / total


def _sequence_kv(s, b):
    """Keys and values of sequence b in float32, [Hk][n][D]."""
    n = s["n"][b][0]
    if s["c"]["op"] == "prompt":
        k0 = s["atk"][b]
        return [s[x][k0:k0 + n].float().view(n, s["c"]["Hk"], -1).transpose(0, 1) for x in "kv"]
    pages = s["table"][b, :s["need"][b]].long()
    out = []
    for x in "kv":
        v = _values(s[x + "q"][pages], s[x + "e"][pages])                              # [pages][Hk][page][D]
        out.append(v.transpose(0, 1).flatten(1, 2)[:, :n])
    return out


def _plain_attention(s):
    c, o = s["c"], s["o"]
    Hq, Hk, D = c["Hq"], c["Hk"], c["D"]
    g = Hq // Hk
    for b, (n, m) in enumerate(s["n"]):
        r0 = s["at"][b]
        k, v = _sequence_kv(s, b)
        q = s["q"][r0:r0 + m].float().view(m, Hk, g, D) * D ** -0.5
        hide = _hidden(n, m, c["window"])
        for h in range(Hk):
            for i in range(g) if m * g * n > 1 << 26 else [slice(0, g)]:               # one head at a time where they are long
                rows = q[:, h, i].reshape(-1, D)
                each = rows.shape[0] // m
                sink = None if s["sinks"] is None else s["sinks"].view(Hk, g)[h, i].reshape(1, -1).expand(m, -1).reshape(-1, 1)
                r = _softmax_times(rows @ k[h].t(), v[h], hide.repeat_interleave(each, 0) if each > 1 else hide, sink)
                o[r0:r0 + m].view(m, Hk, g, D)[:, h, i] = r.view(m, each, D).squeeze(1).to(o.dtype) if not isinstance(i, slice) else r.view(m, g, D).to(o.dtype)
    return {"o": o}


def run(s):
    c = s["c"]
    op = c["op"]
    if not own:
        return _plain_rope(s) if op == "rope" else _plain_cache(s) if op == "cache" else _plain_attention(s)
    qmm = s["qmm"]
    if op == "rope":
        qmm.rope_axes(s["x"], s["y"], s["pos"], s["freq"], s["axis"], c["T"], c["heads"], c["D"], style=c["style"])
        return {"y": s["y"]}
    if op == "cache":
        qmm.kv_write_mxfp4(s["k"], s["v"], s["kv"], s["cu"], s["lens"], s["table"], s["at"][-1])
        qmm.kv_read_mxfp4(s["kv"], s["cu"], s["lens"], s["table"], s["ko"], s["vo"], s["at"][-1])
        return {"k": s["ko"], "v": s["vo"]}
    if op == "attend":
        qmm.attn_kv_mxfp4(s["q"], s["kv"], s["cu"], s["lens"], s["table"], s["o"], s["at"][-1], c["Hq"], c["m"], c["longest"], s["ws"],
                          window=c["window"], sinks=s["sinks"])
    else:
        qmm.attn_prompt_bf16(s["q"], s["k"], s["v"], s["cu"], s["cuk"], s["o"], c["Hq"], c["Hk"], c["D"], window=c["window"], sinks=s["sinks"])
    return {"o": s["o"]}


# ---- what a pass cannot do without ----
def work(c):
    """Inputs, cached keys and values, and results once each; two flops per multiply-add."""
    size = {"f32": 4, "bf16": 2}
    D = c["D"]
    if c["op"] == "rope":
        n = c["T"] * c["heads"] * D
        return {"bytes": n * (size[c["dtype"]] + size[c["out"]]) + 4 * AXES * c["T"] + 5 * c["pairs"], "flops": 6 * c["T"] * c["heads"] * c["pairs"]}
    n = _lengths(c)
    rows = sum(m for _, m in n)
    if c["op"] == "cache":
        v = 2 * rows * c["Hk"] * D
        return {"bytes": int(v * (size[c["dtype"]] + 2 * 17 / 32 + 2)), "flops": 6 * v}
    seen = sum(_visible(length, m, c["window"]) for length, m in n)                     # (row, key) pairs
    keys = sum(min(length, m + c["window"] - 1) if c["window"] else length for length, m in n)
    byte = 17 / 32 if c["op"] == "attend" else 2
    return {"bytes": int(2 * keys * c["Hk"] * D * byte + rows * c["Hq"] * D * (size[c.get("q", "bf16")] + size[c.get("out", "bf16")])),
            "flops": 4 * seen * c["Hq"] * D}


# ---- the same in 64 bits, from the definitions ----
def _mx64(x):
    """The values that MXFP4 holds for x [..][D], float64."""
    v = x.double().unflatten(-1, (-1, 32))
    amax = v.abs().amax(-1, keepdim=True)
    lg = torch.floor(torch.log2(amax.clamp(min=2.0 ** -149)))
    lg = torch.where(torch.exp2(lg) > amax, lg - 1, lg)
    lg = torch.where(torch.exp2(lg + 1) <= amax, lg + 1, lg)
    unit = torch.exp2(torch.clamp(lg - 2, min=-127.0))
    a = v.abs() / unit
    step = 0.5 + 0.5 * (a >= 2) + 1.0 * (a >= 4)
    a = torch.clamp(torch.round(a / step) * step, max=6.0)                 # round: half to even
    return (torch.sign(v) * a * unit).flatten(-2)


def _held64(q, e):
    """float64 values of packed codes with scale bytes."""
    code = torch.empty((*q.shape[:-1], 2 * q.shape[-1]), dtype=torch.uint8, device=q.device)
    code[..., 0::2] = q % 16
    code[..., 1::2] = q // 16
    m = (code % 8).double()
    mag = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8))
    v = torch.where(code >= 8, -mag, mag).unflatten(-1, (-1, 32))
    return (v * torch.exp2(e.double() - 127).unsqueeze(-1)).flatten(-2)


def exact(c, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = kept
    op, D = c["op"], c["D"]
    if op == "rope":
        T, H, P = c["T"], c["heads"], c["pairs"]
        z = s["x"].double().view(T, H, D)
        i = torch.arange(P, device=DEV)
        a, b = (i, i + P) if c["style"] == "halves" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.ones((T, 1, P), dtype=torch.float64, device=DEV),
                           (s["pos"].double()[s["axis"].long(), :].t() * s["freq"].double()).unsqueeze(1))
        w = torch.complex(z[:, :, a], z[:, :, b]) * turn
        z[:, :, a], z[:, :, b] = w.real, w.imag
        return {"y": z.view(T, H * D)}
    if op == "cache":
        return {x: _mx64(s[x].view(-1, c["Hk"], D)).flatten(1) for x in "kv"}
    Hq, Hk = c["Hq"], c["Hk"]
    o = torch.empty((s["at"][-1], Hq, D), dtype=torch.float64, device=DEV)
    for b, (n, m) in enumerate(s["n"]):
        for hk in range(Hk):
            if op == "prompt":
                k, v = (s[x].view(-1, Hk, D)[s["atk"][b]:s["atk"][b + 1], hk].double() for x in "kv")
            else:
                pg = s["table"][b, :s["need"][b]].long()
                k, v = (_held64(s[x + "q"][pg, hk], s[x + "e"][pg, hk]).view(-1, D)[:n] for x in "kv")
            for h in range(hk * Hq // Hk, (hk + 1) * Hq // Hk):
                for i0 in range(0, m, 2048):                                 # rows i0 .. i1, keys up to the last one's
                    i1 = min(m, i0 + 2048)
                    last = n - m + i1
                    l = (s["q"].view(-1, Hq, D)[s["at"][b] + i0:s["at"][b] + i1, h].double() @ k[:last].t()) / math.sqrt(D)
                    p = torch.arange(n - m + i0, last, device=DEV).view(-1, 1)
                    j = torch.arange(last, device=DEV)
                    seen = (j <= p) & (j > p - (c["window"] or n + 1))
                    l = torch.where(seen, l, torch.full_like(l, -math.inf))
                    if c["sinks"]:
                        l = torch.cat([l, s["sinks"][h].double().expand(i1 - i0, 1)], 1)
                    w = torch.softmax(l, 1)[:, :last]
                    o[s["at"][b] + i0:s["at"][b] + i1, h] = w @ v[:last]
    return {"o": o.view(-1, Hq * D)}
