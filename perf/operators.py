"""The operators between a decoder's quantized linears, for a batch of sequences that share a prompt:
the residual's addition with the RMS norm and the quantizer (`mxu.norm_quantize`), attention over a
shared prefix and each sequence's own cache (`attention.shared`), and eviction from that cache by
accumulated attention weight (`attention.evict`).

`run` computes them in their plain form, elementary torch operations in 32 bits, or where `own` is
true calls the framework.  `exact` computes them from their definitions in 64 bits."""
import math

import torch

own = False
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADS = {"Hq": 16, "Hkv": 8, "D": 128}                    # Qwen3-0.6B's and Qwen3-1.7B's heads
EPS = 1e-6


def listed():
    return [
        # one token each for a few sequences on a short system prompt: launches and latency
        {"name": "attn_decode4_1k", "op": "attn", "dt": "bf16", "B": 4, "Lq": 1, **HEADS, "P": 1024, "T": 256,
         "weights": False},
        # a serving batch on a long document, its sums of attention weight kept for eviction
        {"name": "attn_decode64_16k", "op": "attn", "dt": "bf16", "B": 64, "Lq": 1, **HEADS, "P": 16384, "T": 1024,
         "weights": True},
        # the largest batch and prefix
        {"name": "attn_decode256_128k", "op": "attn", "dt": "bf16", "B": 256, "Lq": 1, **HEADS, "P": 131072, "T": 1024,
         "weights": False},
        # eight query heads a cache head of 64, sizes of no round length, fp16
        {"name": "attn_decode23_g8_fp16", "op": "attn", "dt": "fp16", "B": 23, "Lq": 1, "Hq": 24, "Hkv": 3, "D": 64,
         "P": 4099, "T": 517, "weights": True},
        # a draft of seven tokens a sequence checked at once
        {"name": "attn_draft16x7_8k", "op": "attn", "dt": "bf16", "B": 16, "Lq": 7, **HEADS, "P": 8191, "T": 2048,
         "weights": True},
        # pieces of eight prompts after the shared one
        {"name": "attn_prompt8x512_8k", "op": "attn", "dt": "bf16", "B": 8, "Lq": 512, **HEADS, "P": 8192, "T": 1024,
         "weights": False},
        # every sequence one token over its budget, as after each decoded token
        {"name": "evict_step32", "op": "evict", "dt": "bf16", "B": 32, "H": 8, "D": 128, "T": 1040, "n": 1025,
         "budget": 1024, "recent": 64, "ragged": False},
        # caches of several lengths cut to a budget, once in many tokens
        {"name": "evict_batch64", "op": "evict", "dt": "bf16", "B": 64, "H": 8, "D": 128, "T": 2048, "n": 2047,
         "budget": 1000, "recent": 128, "ragged": True},
        # four long prompts cut to an eighth after they were read
        {"name": "evict_prompt4_32k", "op": "evict", "dt": "fp16", "B": 4, "H": 8, "D": 128, "T": 32768, "n": 32768,
         "budget": 4096, "recent": 256, "ragged": False},
        # one decoded token's row in front of a linear
        {"name": "norm_1x1024_fp32", "op": "norm", "dt": "fp32", "M": 1, "K": 1024, "res": True, "row": False},
        # a batch's or a prompt's rows of no round number
        {"name": "norm_509x2048_bf16", "op": "norm", "dt": "bf16", "M": 509, "K": 2048, "res": True, "row": True},
        # many prompts' rows
        {"name": "norm_16384x4096_fp32", "op": "norm", "dt": "fp32", "M": 16384, "K": 4096, "res": True, "row": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case, at most as much work as the largest listed one of its operator."""
    op = rng.choice(["attn", "attn", "attn", "evict", "norm"])
    while True:
        if op == "attn":
            Hkv, G = rng.choice([(1, 8), (2, 4), (3, 5), (4, 1), (8, 2), (8, 4), (16, 1), (2, 16)])
            c = {"op": op, "dt": rng.choice(["bf16", "fp16"]), "B": _log(rng, 1, 256),
                 "Lq": 1 if rng.random() < 0.6 else _log(rng, 2, 512), "Hq": Hkv * G, "Hkv": Hkv,
                 "D": rng.choice([64, 128, 128, 8 * rng.randint(4, 32)]), "P": _log(rng, 100, 131072),
                 "T": _log(rng, 16, 4096), "weights": rng.random() < 0.5}
            rows = c["B"] * c["Lq"] * c["Hq"]
            if c["Lq"] > c["T"] or rows * (c["P"] + c["T"]) > 5.4e8:
                continue
        elif op == "evict":
            n = _log(rng, 64, 32768)
            budget = n - 1 if rng.random() < 0.3 else _log(rng, 16, n)
            c = {"op": op, "dt": rng.choice(["bf16", "fp16"]), "B": _log(rng, 1, 128), "H": rng.randint(1, 8),
                 "D": rng.choice([64, 128, 8 * rng.randint(4, 32)]), "T": n + rng.randint(0, 40), "n": n,
                 "budget": budget, "recent": rng.randint(0, budget // 2), "ragged": rng.random() < 0.5}
        else:
            c = {"op": op, "dt": rng.choice(["bf16", "fp16", "fp32"]), "M": _log(rng, 1, 16384),
                 "K": 32 * _log(rng, 8, 512), "res": rng.random() < 0.8, "row": rng.random() < 0.3}
        top = [work(x) for x in listed() if x["op"] == op]
        w = work(c)
        if all(w[k] <= max(t[k] for t in top) for k in w) and (op != "evict" or _cache_values(c) <= 1.4e8):
            return c


def _cache_values(c):
    return c["B"] * c["T"] * c["H"] * c["D"]


# ---- inputs -----------------------------------------------------------------------------------


def _lens(c, n, least, g):
    """Own lengths of a batch in service: most sequences somewhere up to n, one at n, where there are several one at
    `least`."""
    lens = torch.randint(least, n + 1, (c["B"],), generator=g, device=DEV, dtype=torch.int32)
    lens[0] = n
    if c["B"] > 2:
        lens[1] = least
    return lens


def prepare(case, seed):
    c, g = case, torch.Generator(DEV).manual_seed(seed)
    dt = DT[c["dt"]]

    def rand(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype)

    if c["op"] == "attn":
        B, Lq, Hq, Hkv, D, P, T = (c[k] for k in ("B", "Lq", "Hq", "Hkv", "D", "P", "T"))
        # queries and keys as the norms in front of attention leave them; a few prefix keys draw much of the weight
        pk = rand(P, Hkv, D)
        pk[:4] *= 1.5
        s = {"q": rand(B, Lq, Hq, D) * 1.2, "pk": pk, "pv": rand(P, Hkv, D), "k": rand(B, T, Hkv, D),
             "v": rand(B, T, Hkv, D), "lens": _lens(c, T, Lq, g), "weights": None}
        if c["weights"]:
            s["weights"] = torch.rand((B, Hkv, T), generator=g, device=DEV)
    elif c["op"] == "evict":
        B, H, D, T, n, budget = (c[k] for k in ("B", "H", "D", "T", "n", "budget"))
        s = {"k": rand(B, T, H, D), "v": rand(B, T, H, D),
             "lens": _lens(c, n, max(1, n // 4), g) if c["ragged"] else torch.full((B,), n, dtype=torch.int32, device=DEV)}
        # sums of attention weight: a few tokens hold most, many are alike, the newest have none yet
        w = (rand(B, H, T, dtype=torch.float32) * 2).exp()
        w = torch.where(w < 0.25, torch.floor(w * 64) / 64, w)
        # earlier evictions have left the first slots in no order of their positions
        first = min(budget, n)
        order = torch.rand((B, H, first), generator=g, device=DEV).argsort(-1).to(torch.int32)
        pos = torch.arange(T, device=DEV, dtype=torch.int32).repeat(B, H, 1)
        pos[:, :, :first] = order
        live = torch.arange(T, device=DEV) < s["lens"][:, None, None]
        s["weights"] = torch.where(live, w, 0)
        s["pos"] = torch.where(live, pos, -1)
        # the next step's sums, positions and lengths, kept beside this step's
        s["new"] = (torch.empty_like(w), torch.empty_like(pos), torch.empty_like(s["lens"]))
    else:
        M, K = c["M"], c["K"]
        s = {"x": rand(M, K), "res": None, "gamma": 1 + 0.2 * rand(K, dtype=torch.float32)}
        if c["res"]:
            # a residual stream: rows of several sizes, a few columns far above the others
            r = rand(M, K, dtype=torch.float32) * (0.5 + 3 * torch.rand((M, 1), generator=g, device=DEV))
            r[:, :: max(1, K // 5)] *= 12
            s["res"] = r.to(dt)
    s["case"] = c
    return s


# ---- one pass ---------------------------------------------------------------------------------


def _plain_attn(s, c):
    B, Lq, Hkv, D, P, T = (c[k] for k in ("B", "Lq", "Hkv", "D", "P", "T"))
    R = Lq * (c["Hq"] // Hkv)                              # rows of a sequence and cache head: (token, query head)
    q = (s["q"].float() * D ** -0.5).view(B, Lq, Hkv, -1, D).permute(2, 0, 1, 3, 4).reshape(Hkv, B * R, D)
    pk, pv = s["pk"].float().transpose(0, 1), s["pv"].float().transpose(0, 1)
    k, v = s["k"].float().permute(2, 0, 1, 3), s["v"].float().permute(2, 0, 1, 3)
    sp = torch.matmul(q, pk.transpose(1, 2)).view(Hkv, B, R, P)
    so = torch.matmul(q.view(Hkv, B, R, D), k.transpose(2, 3))
    at = s["lens"][:, None] - Lq + torch.arange(Lq, device=DEV)
    hidden = torch.arange(T, device=DEV) > at[:, :, None]  # [B, Lq, T]
    so = so.view(Hkv, B, Lq, -1, T).masked_fill_(hidden[None, :, :, None], -math.inf).view(Hkv, B, R, T)
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    sp, so = sp.sub_(m).exp_(), so.sub_(m).exp_()
    l = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    o = torch.matmul(sp.view(Hkv, B * R, P), pv).view(Hkv, B, R, D) + torch.matmul(so, v)
    o = (o / l).view(Hkv, B, Lq, -1, D).permute(1, 2, 0, 3, 4).reshape(B, Lq, -1, D).to(s["q"].dtype)
    if s["weights"] is None:
        return {"out": o}
    s["weights"] += (so / l).sum(2).transpose(0, 1)
    return {"out": o, "weights": s["weights"]}


def _plain_evict(s, c):
    B, H, D, T, budget = (c[k] for k in ("B", "H", "D", "T", "budget"))
    w, pos = s["weights"], s["pos"]
    t = torch.arange(T, device=DEV)
    n = s["lens"][:, None, None]
    left = n.clamp(max=budget)
    safe = pos > pos.amax(-1, keepdim=True) - c["recent"]
    key = torch.where(t < n, torch.where(safe, math.inf, w), -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, order, (t < left).expand(B, H, T))
    hole, extra = (t < left) & ~keep, (t >= left) & keep
    sources = (~extra).to(torch.int8).sort(dim=-1, stable=True).indices       # kept slots past the budget, in order
    src = torch.where(hole, sources.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), t)
    s["new"][0].copy_(torch.where(t < left, w.gather(-1, src), 0))
    s["new"][1].copy_(torch.where(t < left, pos.gather(-1, src), -1))
    s["new"][2].copy_(s["lens"].clamp(max=budget))
    at = src[:, :, :budget].transpose(1, 2)[..., None].expand(B, -1, H, D)
    s["k"][:, :budget] = s["k"].gather(1, at)
    s["v"][:, :budget] = s["v"].gather(1, at)
    return {"weights": s["new"][0], "pos": s["new"][1], "lens": s["new"][2], "k": s["k"], "v": s["v"]}


def _values(q, d):
    """The operand's values over its row's scale, q 2^-d: seven bits and a power of two, whole in bfloat16."""
    q = q.view(*d.shape, 32)
    return torch.mul(q, torch.pow(0.5, d)[..., None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=DEV))


def _plain_norm(s, c):
    h = s["x"].float()
    if s["res"] is not None:
        h = h + s["res"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["gamma"]
    groups = y.view(c["M"], -1, 32)
    amax = groups.abs().amax(-1)
    top = amax.amax(-1, keepdim=True)
    if c["row"]:
        d = torch.zeros_like(amax)
    else:                                                  # the largest d with amax_g 2^d <= amax
        (fm, fe), (gm, ge) = torch.frexp(top), torch.frexp(amax)
        d = torch.where(amax > 0, (fe - ge - (gm > fm).int()).clamp(0, 31), 0)
    q = torch.round(groups * (127 / top * torch.exp2(d.float()))[..., None]).clamp(-127, 127)
    out = {"values": _values(q, d), "S": (top / 127)[:, 0]}
    if s["res"] is not None:
        out["h"] = h.to(s["x"].dtype)
    return out


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"attn": _plain_attn, "evict": _plain_evict, "norm": _plain_norm}[c["op"]](s, c)
    from opentpu_amd import attention, mxu
    if c["op"] == "attn":
        o = attention.shared(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lens"], weights=s["weights"])
        return {"out": o} if s["weights"] is None else {"out": o, "weights": s["weights"]}
    if c["op"] == "evict":
        w, pos, lens = attention.evict(s["k"], s["v"], s["weights"], s["pos"], s["lens"], c["budget"], c["recent"],
                                       out=s["new"])
        return {"weights": w, "pos": pos, "lens": lens, "k": s["k"], "v": s["v"]}
    op, h = mxu.norm_quantize(s["x"], s["gamma"], s["res"], eps=EPS, row_mode=c["row"])
    q, S, d, _ = op
    out = {"values": _values(q, d), "S": S[0]}
    if s["res"] is not None:
        out["h"] = h
    return out


def work(case):
    c = case
    e = 4 if c["dt"] == "fp32" else 2
    if c["op"] == "attn":
        n = c["B"] * (c["Lq"] + c["T"]) / 2                # own tokens of the batch, in the mean
        rows = c["B"] * c["Lq"] * c["Hq"]
        b = e * c["D"] * (2 * rows + 2 * c["Hkv"] * (c["P"] + n)) + (8 * c["Hkv"] * n if c["weights"] else 0)
        return {"bytes": b, "flops": 4 * c["D"] * rows * (c["P"] + max(1, (c["T"] - c["Lq"]) / 2 + c["Lq"] / 2))}
    if c["op"] == "evict":
        n = c["n"] * (0.625 if c["ragged"] else 1)
        moved = max(1, c["budget"] * (n - c["budget"]) / n) if n > c["budget"] else 0
        slots = c["B"] * c["H"]
        return {"bytes": slots * (16 * c["T"] + 4 * e * c["D"] * moved), "flops": slots * n}
    n = c["M"] * c["K"]
    return {"bytes": n * (e * (3 if c["res"] else 1) + 1 + 1 / 32) + 4 * c["M"] + 4 * c["K"], "flops": 12 * n}


# ---- the definitions in 64 bits ---------------------------------------------------------------


def _exact_attn(s, c):
    B, Lq, Hq, Hkv, D, P = (c[k] for k in ("B", "Lq", "Hq", "Hkv", "D", "P"))
    G, lens = Hq // Hkv, s["lens"].tolist()
    q = s["q"].double() / math.sqrt(D)
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    w = None if s["weights"] is None else s["weights"].double()
    for h in range(Hkv):
        qh = q[:, :, h * G:(h + 1) * G]
        sp = qh.reshape(-1, D) @ s["pk"][:, h].double().T
        lse_p = torch.logsumexp(sp, -1)
        op = (sp.sub_(lse_p[:, None]).exp_() @ s["pv"][:, h].double()).view(B, Lq, G, D)
        lse_p = lse_p.view(B, Lq, G)
        for b in range(B):
            n = lens[b]
            so = (qh[b].reshape(-1, D) @ s["k"][b, :n, h].double().T).view(Lq, G, n)
            seen = torch.ones((Lq, n), dtype=torch.bool, device=DEV).tril(n - Lq)
            so = so.masked_fill(~seen[:, None], -math.inf)
            lse = torch.logaddexp(lse_p[b], torch.logsumexp(so, -1))
            p = torch.exp(so - lse[..., None])
            o = op[b] * torch.exp(lse_p[b] - lse)[..., None] + (p.view(-1, n) @ s["v"][b, :n, h].double()).view(Lq, G, D)
            out[b, :, h * G:(h + 1) * G] = o
            if w is not None:
                w[b, h, :n] += p.sum((0, 1))
    return {"out": out} if w is None else {"out": out, "weights": w}


def _exact_evict(s, c):
    budget, lens = c["budget"], s["lens"].tolist()
    w, pos = s["weights"].cpu(), s["pos"].cpu()
    nw, npos = torch.zeros_like(w, dtype=torch.float64), torch.full_like(pos, -1)
    for b, n in enumerate(lens):
        left = min(n, budget)
        for h in range(c["H"]):
            wb, pb = w[b, h, :n].tolist(), pos[b, h, :n].tolist()
            last = max(pb) - c["recent"]
            kept = sorted(range(n), key=lambda t: (pb[t] <= last, 0.0 if pb[t] > last else -wb[t], t))[:left]
            stay = set(t for t in kept if t < left)
            src = list(range(left))
            for t, u in zip((t for t in range(left) if t not in stay), sorted(t for t in kept if t >= left)):
                src[t] = u
            nw[b, h, :left] = torch.tensor([wb[t] for t in src], dtype=torch.float64)
            npos[b, h, :left] = torch.tensor([pb[t] for t in src], dtype=torch.int32)
            at = torch.tensor(src, device=DEV)
            for x in (s["k"], s["v"]):
                x[b, :left, h] = x[b, at, h]
    return {"weights": nw, "pos": npos, "lens": torch.tensor([min(n, budget) for n in lens], dtype=torch.int32),
            "k": s["k"], "v": s["v"]}


def _exact_norm(s, c):
    h = s["x"].double() + (s["res"].double() if s["res"] is not None else 0)
    y = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + EPS) * s["gamma"].double()
    y = y.view(c["M"], c["K"] // 32, 32)
    S = y.abs().amax((1, 2)) / 127
    step = S[:, None, None].expand(-1, c["K"] // 32, 1)
    if not c["row"]:
        d = torch.floor(torch.log2(S[:, None] * 127 / y.abs().amax(-1))).clamp(0, 31)
        step = step / torch.exp2(d)[..., None]
    out = {"values": torch.round(y / step).clamp(-127, 127) * step / S[:, None, None], "S": S}
    if s["res"] is not None:
        out["h"] = h
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "evict": _exact_evict, "norm": _exact_norm}[case["op"]](s, case)
