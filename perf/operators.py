"""The operators of an MXFP4 decoder block, as measurable cases: what one call of each reads and answers, in
plain torch (own = False) and through hipster_amd.qmm (own = True).

ops
  route     a token's experts from its router logits: softmax or sigmoid scores, a balance bias, groups of
            experts, top-k, renormalised and scaled weights, the shared expert's slot
  mxfp4     rows quantised to MXFP4 (blocks of 32 values, one power-of-two scale) and read back as values
  product   activations quantised to MXFP4, then times an MXFP4 weight: decode GEMV up to 64 rows, GEMM beyond
  experts   activations quantised to MXFP4, then every token's row times its experts' MXFP4 weights: by the
            routed ids up to 16 tokens, over rows sorted by expert beyond
  norm      the norm after a block, its gate, the scaled residual addition and the next block's norm

Sizes are those of hipster_amd.synth and bench.py (a dense 5120 / 17408 model, a 512-expert 2048 / 512 MoE) and
generic ones.  Weights are normal numbers of deviation 1 / sqrt(K) quantised to MXFP4; activations are normal with
a few channels sixteen times larger, as trained models have them.
"""
import numpy as np
import torch

own = False

EPS = 1e-6
DEV = "cuda"
GEMV_ROWS, MOE_GEMV_TOKENS = 64, 16      # the longest calls of the decode forms
TILE_ROWS = 128                          # rows of one expert in a tile of the sorted form


def listed():
    return [
        # one user's decode step: 512 softmax scores, top 10 and the shared expert; nothing but latency
        dict(name="route_t1", op="route", T=1, E=512, k=10, score="softmax", bias=False, groups=1, keep=1, best=1, renorm=True,
             scale=1.0, shared=True),
        # a long prompt: sigmoid scores with a balance bias, 4 of 8 groups by their two best, top 8
        dict(name="route_t4096", op="route", T=4096, E=256, k=8, score="sigmoid", bias=True, groups=8, keep=4, best=2, renorm=True,
             scale=2.5, shared=False),
        # the activations of a few drafted tokens, f32, rows that end inside a block of 128
        dict(name="mxfp4_r5", op="mxfp4", R=5, K=2880, dtype="f32"),
        # a prompt chunk's MLP activations, bf16
        dict(name="mxfp4_r2048", op="mxfp4", R=2048, K=17408, dtype="bf16"),
        # one user's decode step through an MLP's gate or up projection
        dict(name="product_m1", op="product", M=1, N=17408, K=5120, dtype="bf16", out="f32"),
        # a batch of 24 users through the down projection
        dict(name="product_m24", op="product", M=24, N=5120, K=17408, dtype="f32", out="f32"),
        # a prompt of ordinary, ragged length
        dict(name="product_m300", op="product", M=300, N=17408, K=5120, dtype="bf16", out="bf16"),
        # a full prompt chunk: the largest call
        dict(name="product_m2048", op="product", M=2048, N=17408, K=5120, dtype="bf16", out="bf16"),
        # a decode step of four users through the 512-expert MoE: gate and up rows as one weight
        dict(name="experts_t4", op="experts", T=4, E=512, k=10, shared=True, N=1024, K=2048, dtype="bf16", out="f32"),
        # a full prompt chunk through it: some 44 rows an expert, the weights' bytes decide
        dict(name="experts_t2048", op="experts", T=2048, E=512, k=10, shared=True, N=1024, K=2048, dtype="bf16", out="bf16"),
        # one user's decode step between two blocks
        dict(name="norm_t1", op="norm", T=1, n=5120, y="f32", post=True, gate="token", act="sigmoid", alpha=0.22),
        # a full prompt chunk between two blocks, a gate for every value
        dict(name="norm_t2048", op="norm", T=2048, n=5120, y="bf16", post=True, gate="value", act="silu", alpha=1.0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "mxfp4", "product", "product", "product", "experts", "experts", "norm"])
    if op == "route":
        E = rng.choice([8, 60, 64, 128, 160, 256, 384, 512])
        groups = rng.choice([1, 1, 2, 4, 8]) if E % 8 == 0 else 1
        keep = rng.randint(max(1, groups // 2), groups)
        k = min(rng.choice([1, 2, 4, 6, 8, 10]), keep * (E // groups))
        return dict(op=op, T=_spread(rng, 1, 8192), E=E, k=k, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    groups=groups, keep=keep, best=rng.choice([1, 2]) if E // groups > 1 else 1, renorm=rng.random() < 0.8,
                    scale=rng.choice([1.0, 2.5]), shared=rng.random() < 0.5)
    if op == "mxfp4":
        K = _spread(rng, 32, 17408)
        return dict(op=op, R=_spread(rng, 1, max(1, min(8192, 2048 * 17408 // K))), K=K, dtype=rng.choice(["f32", "bf16"]))
    if op == "norm":
        n = 32 * _spread(rng, 8, 256) + rng.choice([0, 0, 0, 4, 7])
        return dict(op=op, T=_spread(rng, 1, 4096), n=n, y=rng.choice(["f32", "bf16"]), post=rng.random() < 0.7,
                    gate=rng.choice(["none", "token", "channel", "value"]), act=rng.choice(["none", "sigmoid", "silu"]),
                    alpha=rng.choice([1.0, 0.22]))
    odd = lambda v: v if rng.random() < 0.6 else v + rng.randint(1, 63)      # noqa: E731
    if op == "product":
        N, K = odd(_spread(rng, 256, 17300)), odd(_spread(rng, 256, 17300))
        room = 2048 * 17408 * 5120 // (N * K)
        return dict(op=op, M=min(_spread(rng, 1, 2048), room), N=N, K=K, dtype=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]))
    E = rng.choice([16, 64, 128, 256, 512])
    return dict(op=op, T=_spread(rng, 1, 2048), E=E, k=rng.choice([2, 4, 8, 10]), shared=rng.random() < 0.5, N=odd(_spread(rng, 128, 1000)),
                K=odd(_spread(rng, 128, 2000)), dtype=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]))


# ---- the MXFP4 format in plain torch ----
def _pow2(e):
    """2^e for whole e in float64, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantise(x):
    """Rows [R][K] -> codes [R][K] (uint8: sign and three bits) and scale bytes [R][ceil(K / 32)]."""
    R, K = x.shape
    nb = -(-K // 32)
    v = torch.zeros((R, nb * 32), dtype=torch.float32, device=x.device)
    v[:, :K] = x.float()
    v = v.view(R, nb, 32)
    amax = v.abs().amax(2)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, torch.full_like(amax, -127, dtype=torch.int32)).clamp(min=-127)
    t = (v.double() * _pow2(-e).unsqueeze(2)).abs().float()
    code = (t > 0.25).byte()
    for border, closed in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (t >= border) if closed else (t > border)
    code |= torch.signbit(v).byte() << 3
    return code.view(R, nb * 32)[:, :K], (e + 127).byte()


def _values(code, scale):
    """float32 values of codes [.., K] with scale bytes [.., ceil(K / 32)]."""
    K = code.shape[-1]
    level = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    s = _pow2(scale.int() - 127).float()
    return level[code.long()] * s.repeat_interleave(32, -1)[..., :K]


def _pack(code):
    """Codes [R][K] -> bytes [R][64 * ceil(K / 128)], the even value in the low half, padded with zeros."""
    R, K = code.shape
    p = torch.zeros((R, -(-K // 128) * 128), dtype=torch.uint8, device=code.device)
    p[:, :K] = code
    return p[:, 0::2] | (p[:, 1::2] << 4)


def _unpack(q, K):
    return torch.stack([q & 15, q >> 4], -1).flatten(-2)[..., :K]


def _pad_scales(e):
    """Scale bytes [R][nb] -> [R][4 * ceil(nb / 4)], padded with zeros."""
    p = torch.zeros((e.shape[0], -(-e.shape[1] // 4) * 4), dtype=torch.uint8, device=e.device)
    p[:, :e.shape[1]] = e
    return p


# ---- inputs ----
_T = {"f32": torch.float32, "bf16": torch.bfloat16}


def _rows(g, R, K, dtype):
    x = torch.randn((R, K), device=DEV, generator=g)
    big = torch.randint(0, K, (max(1, K // 256),), device=DEV, generator=g)
    x[:, big] *= 16.0
    return x.to(_T[dtype])


def _weights(g, n, K):
    """n rows of K MXFP4 weights: packed bytes and padded scale bytes."""
    q, e = [], []
    step = max(1, (1 << 27) // K)
    for i in range(0, n, step):
        code, sc = _quantise(torch.randn((min(step, n - i), K), device=DEV, generator=g) * K ** -0.5)
        q.append(_pack(code))
        e.append(_pad_scales(sc))
    return torch.cat(q), torch.cat(e)


def _routing(g, c):
    """ids [T][slots] (-1 in the last slot for the shared expert) and the rows sorted by expert: token and tiles."""
    T, E, k = c["T"], c["E"], c["k"]
    slots = k + c["shared"]
    ids = torch.full((T, slots), -1, dtype=torch.int32, device=DEV)
    ids[:, :k] = torch.rand((T, E), device=DEV, generator=g).topk(k, 1)[1].int()
    key = torch.where(ids < 0, E, ids.long()).flatten()
    order = torch.sort(key, stable=True)[1]
    n = torch.bincount(key, minlength=E + 1).tolist()
    segs, tiles, k0 = [], [], 0
    for ex, m in enumerate(n):
        if m:
            segs.append((ex if ex < E else -1, k0, k0 + m))
            tiles += [(ex if ex < E else -1, k0 + i, min(TILE_ROWS, m - i)) for i in range(0, m, TILE_ROWS)]
            k0 += m
    return ids, order, segs, tiles


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    op, s = c["op"], dict(c=c)
    empty = lambda *shape, t="f32": torch.empty(shape, dtype=_T[t], device=DEV)      # noqa: E731
    if op == "route":
        T, E, slots = c["T"], c["E"], c["k"] + c["shared"]
        s.update(logits=torch.randn((T, E + c["shared"]), device=DEV, generator=g),
                 bias=torch.randn(E, device=DEV, generator=g) * 0.1 if c["bias"] else None,
                 ids=torch.empty((T, slots), dtype=torch.int32, device=DEV), w=empty(T, slots))
        return s
    if op == "norm":
        T, n = c["T"], c["n"]
        shape = {"none": None, "token": (T, 1), "channel": (n,), "value": (T, n)}[c["gate"]]
        s.update(x=torch.randn((T, n), device=DEV, generator=g) * 4.0, y=_rows(g, T, n, c["y"]),
                 wy=1 + 0.1 * torch.randn(n, device=DEV, generator=g) if c["post"] else None,
                 gate=torch.randn(shape, device=DEV, generator=g).to(_T[c["y"]]) if shape else None,
                 w=1 + 0.1 * torch.randn(n, device=DEV, generator=g), xo=empty(T, n), xb=empty(T, n, t="bf16"))
        return s
    if op == "mxfp4":
        s.update(x=_rows(g, c["R"], c["K"], c["dtype"]), v=empty(c["R"], c["K"], t="bf16"))
        rows, K = c["R"], c["K"]
    else:
        rows, N, K = c["M" if op == "product" else "T"], c["N"], c["K"]
        s.update(x=_rows(g, rows, K, c["dtype"]))
        if op == "experts":
            ids, order, segs, tiles = _routing(g, c)
            s.update(ids=ids, order=order, segs=segs, y=empty(ids.numel(), N, t=c["out"]))
            if not own:
                s["rowtok"] = torch.div(order, ids.shape[1], rounding_mode="floor")
        else:
            s.update(y=empty(rows, N, t=c["out"]))
        q, e = _weights(g, N * (c["E"] + c["shared"] if op == "experts" else 1), K)      # the shared expert last
        if not own:
            s.update(Wq=q.view(-1, N, q.shape[1]), We=e.view(-1, N, e.shape[1]))
    if own:
        from hipster_amd import qmm
        s.update(qmm=qmm, xq=qmm.XMXBuf(rows, K))
        if op == "experts":
            s["eb"] = qmm.mxfp4_weight_bytes(N, K)
            s["W"] = torch.empty((c["E"] + c["shared"], s["eb"]), dtype=torch.uint8, device=DEV)
            for i in range(len(s["W"])):
                qmm.pack_mxfp4(q[i * N:(i + 1) * N], e[i * N:(i + 1) * N], s["W"][i], N, K)
            s["Wsh"] = s["W"][c["E"]] if c["shared"] else None
            s["rowtab"] = torch.div(order, ids.shape[1], rounding_mode="floor").int()
            s["tiles"] = torch.tensor(tiles, dtype=torch.int32, device=DEV)
            routed = sum(t[0] >= 0 for t in tiles)
            s["counts"] = torch.tensor([routed, len(tiles) - routed], dtype=torch.int32, device=DEV)
        elif op == "product":
            s["W"] = torch.empty(qmm.mxfp4_weight_bytes(N, K), dtype=torch.uint8, device=DEV)
            qmm.pack_mxfp4(q, e, s["W"], N, K)
    return s


# ---- one pass, plain ----
def _act(name, v):
    return v if name == "none" else torch.sigmoid(v) if name == "sigmoid" else v * torch.sigmoid(v)


def _plain_route(s):
    c = s["c"]
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    l = s["logits"].double()                      # 64 bits: a choice between two scores is no matter of rounding
    if c["score"] == "softmax":
        p = torch.exp(l[:, :E] - l[:, :E].amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-l[:, :E]))
    choice = p if s["bias"] is None else p + s["bias"].double()
    if c["keep"] < G:
        by_group = torch.sort(choice.view(T, G, E // G), dim=2, descending=True)[0][:, :, :c["best"]].sum(2)
        kept = torch.sort(by_group, dim=1, descending=True, stable=True)[1][:, :c["keep"]]
        mask = torch.zeros((T, G), dtype=torch.bool, device=DEV).scatter_(1, kept, True)
        choice = choice.masked_fill(~mask.repeat_interleave(E // G, 1), -float("inf"))
    ids = torch.sort(choice, dim=1, descending=True, stable=True)[1][:, :k]
    w = p.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = w * c["scale"]
    if c["shared"]:
        ids = torch.cat([ids, torch.full_like(ids[:, :1], -1)], 1)
        w = torch.cat([w, 1.0 / (1.0 + torch.exp(-l[:, E:]))], 1)
    return {"ids": ids.int(), "w": w.float()}


def _plain_experts(s):
    c = s["c"]
    a, y = _values(*_quantise(s["x"])), s["y"]
    rows = a[s["rowtok"]]
    out = y if c["T"] > MOE_GEMV_TOKENS else torch.empty_like(y)
    for first in range(0, len(s["segs"]), 32):                   # the weights of 32 experts at a time
        part = s["segs"][first:first + 32]
        ex = torch.tensor([e for e, _, _ in part], device=DEV)
        W = _values(_unpack(s["Wq"][ex], c["K"]), s["We"][ex])
        for i, (_, k0, k1) in enumerate(part):
            out[k0:k1] = (rows[k0:k1] @ W[i].t()).to(y.dtype)
    if c["T"] <= MOE_GEMV_TOKENS:                                # the decode form answers slot by slot
        y[s["order"]] = out
    return {"y": y}


def _plain_norm(s):
    c = s["c"]
    p = s["y"].float()
    if c["post"]:
        p = p * torch.rsqrt((p * p).mean(1, keepdim=True) + EPS) * s["wy"]
    if s["gate"] is not None:
        p = p * _act(c["act"], s["gate"].float())
    xo = s["x"] + c["alpha"] * p
    return {"x": xo, "xn": (xo * torch.rsqrt((xo * xo).mean(1, keepdim=True) + EPS) * s["w"]).bfloat16()}


def run(s):
    c = s["c"]
    op = c["op"]
    if not own:
        if op == "route":
            return _plain_route(s)
        if op == "norm":
            return _plain_norm(s)
        if op == "experts":
            return _plain_experts(s)
        if op == "mxfp4":
            return {"v": _values(*_quantise(s["x"])).bfloat16()}
        W = _values(_unpack(s["Wq"][0], c["K"]), s["We"][0])
        return {"y": (_values(*_quantise(s["x"])) @ W.t()).to(_T[c["out"]])}
    if op == "norm":
        from hipster_amd import qmm
        qmm.postnorm_add_rmsnorm_bf16(s["x"], s["y"], s["wy"], s["w"], s["xb"], c["T"], c["n"], EPS, gate=s["gate"], act=c["act"],
                                      alpha=c["alpha"], xo=s["xo"])
        return {"x": s["xo"], "xn": s["xb"]}
    if op == "route":
        from hipster_amd import qmm
        qmm.moe_route_groups(s["logits"], s["ids"], s["w"], c["T"], c["E"], c["k"], score=c["score"], bias=s["bias"], groups=c["groups"],
                             keep=c["keep"], best=c["best"], renorm=c["renorm"], scale=c["scale"],
                             shared="gate" if c["shared"] else None)
        return {"ids": s["ids"], "w": s["w"]}
    qmm, xq, K = s["qmm"], s["xq"], c["K"]
    if op == "mxfp4":
        qmm.quantize_mxfp4(s["x"], xq, c["R"], K)
        qmm.dequant_mxfp4(xq, s["v"], c["R"], K)
        return {"v": s["v"]}
    rows = c["M" if op == "product" else "T"]
    qmm.quantize_mxfp4(s["x"], xq, rows, K)
    if op == "product":
        (qmm.gemv_mxfp4 if rows <= GEMV_ROWS else qmm.gemm_mxfp4)(s["W"], xq, s["y"], rows, c["N"], K)
    elif rows <= MOE_GEMV_TOKENS:
        qmm.gemv_moe_mxfp4(s["W"], s["Wsh"], s["eb"], s["ids"], xq, s["y"], rows, s["ids"].shape[1], c["E"], c["N"], K)
    else:
        qmm.moe_gemm_mxfp4(s["W"], s["Wsh"], s["eb"], s["tiles"], s["counts"], len(s["tiles"]), s["rowtab"], xq, s["y"], c["N"], K)
    return {"y": s["y"]}


# ---- what a pass cannot do without ----
def work(c):
    """Inputs, weights and results once each; two flops per multiply-add, a handful per value elsewhere."""
    op = c["op"]
    size = {"f32": 4, "bf16": 2}
    if op == "route":
        return {"bytes": 4 * c["T"] * (c["E"] + c["shared"]) + 8 * c["T"] * (c["k"] + c["shared"]), "flops": 8 * c["T"] * c["E"]}
    if op == "norm":
        gate = {"none": 0, "token": c["T"], "channel": c["n"], "value": c["T"] * c["n"]}[c["gate"]]
        return {"bytes": c["T"] * c["n"] * (4 + size[c["y"]] + 4 + 2) + gate * size[c["y"]] + 8 * c["n"], "flops": 12 * c["T"] * c["n"]}
    K = c["K"]
    if op == "mxfp4":
        return {"bytes": c["R"] * K * (size[c["dtype"]] + 17 / 32 + 2), "flops": 6 * c["R"] * K}
    N = c["N"]
    if op == "product":
        return {"bytes": c["M"] * K * size[c["dtype"]] + N * K * 17 / 32 + c["M"] * N * size[c["out"]], "flops": 2 * c["M"] * N * K}
    T, slots = c["T"], c["k"] + c["shared"]
    reached = c["E"] * (1 - (1 - c["k"] / c["E"]) ** T) + c["shared"]      # the experts that T tokens reach, expected
    return {"bytes": T * K * size[c["dtype"]] + reached * N * K * 17 / 32 + T * slots * N * size[c["out"]], "flops": 2 * T * slots * N * K}


# ---- the same in 64 bits, from the definitions ----
def _mx64(x):
    """The values that MXFP4 holds for the rows x, float64."""
    R, K = x.shape
    pad = -K % 32
    v = torch.nn.functional.pad(x.double(), (0, pad)).view(R, -1, 32)
    amax = v.abs().amax(2, keepdim=True)
    lg = torch.floor(torch.log2(amax.clamp(min=2.0 ** -149)))
    lg = torch.where(torch.exp2(lg) > amax, lg - 1, lg)
    lg = torch.where(torch.exp2(lg + 1) <= amax, lg + 1, lg)
    unit = torch.exp2(torch.clamp(lg - 2, min=-127.0))
    a = v.abs() / unit
    step = 0.5 + 0.5 * (a >= 2) + 1.0 * (a >= 4)
    a = torch.clamp(torch.round(a / step) * step, max=6.0)                 # round: half to even
    return (torch.sign(v) * a * unit).view(R, -1)[:, :K]


def _held64(q, e, K):
    """float64 values of packed rows."""
    code = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.uint8, device=q.device)
    code[:, 0::2] = q % 16
    code[:, 1::2] = q // 16
    m = (code % 8).double()
    mag = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8))
    v = torch.where(code >= 8, -mag, mag).view(q.shape[0], -1, 32)
    return (v * torch.exp2(e.double() - 127).unsqueeze(2)).view(q.shape[0], -1)[:, :K]


def _route64(c, logits, bias):
    l = logits.double().cpu().numpy()
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    z = l[:, :E]
    if c["score"] == "softmax":
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 1 / (1 + np.exp(-z))
    choice = p + (0 if bias is None else bias.double().cpu().numpy())
    ids = np.empty((T, k + c["shared"]), np.int32)
    w = np.empty((T, k + c["shared"]))
    for t in range(T):
        members = np.arange(E).reshape(G, E // G)
        if c["keep"] < G:
            value = [np.sort(choice[t, m])[::-1][:c["best"]].sum() for m in members]
            members = members[np.lexsort((np.arange(G), -np.array(value)))[:c["keep"]]]
        cand = np.sort(members.ravel())
        sel = cand[np.lexsort((cand, -choice[t, cand]))[:k]]
        ids[t, :k] = sel
        w[t, :k] = p[t, sel] / (p[t, sel].sum() if c["renorm"] else 1.0) * c["scale"]
        if c["shared"]:
            ids[t, k], w[t, k] = -1, 1 / (1 + np.exp(-l[t, E]))
    return {"ids": torch.from_numpy(ids).to(DEV), "w": torch.from_numpy(w).to(DEV)}


def exact(c, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = kept
    op = c["op"]
    if op == "route":
        return _route64(c, s["logits"], s["bias"])
    if op == "mxfp4":
        return {"v": _mx64(s["x"])}
    if op == "norm":
        rms = lambda v: v / torch.sqrt((v ** 2).sum(1, keepdim=True) / c["n"] + EPS)      # noqa: E731
        p = s["y"].double()
        if c["post"]:
            p = rms(p) * s["wy"].double()
        if s["gate"] is not None:
            z = s["gate"].double()
            p = p * {"none": z, "sigmoid": 1 / (1 + torch.exp(-z)), "silu": z / (1 + torch.exp(-z))}[c["act"]]
        xo = s["x"].double() + c["alpha"] * p
        return {"x": xo, "xn": rms(xo) * s["w"].double()}
    a = _mx64(s["x"])
    if op == "product":
        return {"y": a @ _held64(s["Wq"][0], s["We"][0], c["K"]).t()}
    ids = s["ids"].flatten().long()
    tok = torch.arange(len(ids), device=DEV) // s["ids"].shape[1]
    y = torch.empty((len(ids), c["N"]), dtype=torch.float64, device=DEV)
    for ex in torch.unique(ids).tolist():
        at = torch.nonzero(ids == ex).flatten()
        y[at] = a[tok[at]] @ _held64(s["Wq"][ex], s["We"][ex], c["K"]).t()
    return {"y": y if c["T"] <= MOE_GEMV_TOKENS else y[s["order"]]}
