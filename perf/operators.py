"""Workloads for the mixture-of-experts operators (kernels.moe_route, moe_experts, moe_layer) and the several-axis rotary
embedding with its paged cache write (kernels.qkv_mrope_kv_write): named cases, drawn cases of the same ranges, inputs,
one pass through the framework's call or through the same formula in elementary torch operations, and the formula in 64
bits.

The largest cases are long prompts (thousands of tokens, where the experts' weights are read once for many tokens); the
smallest are single decode steps, where latency counts.
"""
from __future__ import annotations

import math

import torch

own = False

BF16 = torch.bfloat16
FLT_MAX = torch.finfo(torch.float32).max


# ----------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # routing of one decode batch: 256 experts, 8 a token and a shared one, bf16 logits (ties are common)
        {"name": "route decode", "op": "route", "T": 64, "E": 256, "k": 8, "shared": True, "renorm": True,
         "f32": False, "masked": False},
        # routing of a long prompt with fp32 logits; experts outside a token's allowed set at -inf, padding rows all -inf
        {"name": "route prompt", "op": "route", "T": 16384, "E": 160, "k": 6, "shared": False, "renorm": False,
         "f32": True, "masked": True},
        # a single user's decode step: nine experts' weights, latency
        {"name": "layer one token", "op": "layer", "T": 1, "E": 256, "k": 8, "H": 2048, "I": 512, "shared": True},
        # speculative or small-batch decode, an odd number of rows
        {"name": "layer small batch", "op": "layer", "T": 7, "E": 256, "k": 8, "H": 2048, "I": 512, "shared": True},
        # a decode batch: most experts are hit by a few tokens each, every weight is read
        {"name": "layer decode", "op": "layer", "T": 64, "E": 256, "k": 8, "H": 2048, "I": 512, "shared": True},
        # few large experts, two a token, at decode
        {"name": "experts decode large", "op": "experts", "T": 32, "E": 8, "k": 2, "H": 4096, "I": 7168, "pad": 0},
        # a chunk of a prompt: tens of tokens an expert; ragged sizes, the last rows are padding
        {"name": "experts chunk", "op": "experts", "T": 777, "E": 60, "k": 4, "H": 2048, "I": 1408, "pad": 9},
        # a prompt: every expert over a hundred tokens
        {"name": "experts prompt", "op": "experts", "T": 4096, "E": 256, "k": 8, "H": 2048, "I": 512, "pad": 0},
        # few large experts on a prompt: bound by the products
        {"name": "experts prompt large", "op": "experts", "T": 4096, "E": 8, "k": 2, "H": 4096, "I": 7168, "pad": 0},
        # one decode step: rotate and append 64 rows
        {"name": "mrope decode", "op": "mrope", "T": 64, "nq": 16, "nkv": 2, "hd": 128, "rd": 128, "axes": 3,
         "interleaved": True, "block": 16, "pad": 0},
        # an image prompt with a partial rotation, odd length, padding rows
        {"name": "mrope partial", "op": "mrope", "T": 1777, "nq": 16, "nkv": 2, "hd": 256, "rd": 64, "axes": 3,
         "interleaved": True, "block": 64, "pad": 5},
        # a long video prompt, sections in blocks
        {"name": "mrope video", "op": "mrope", "T": 16384, "nq": 32, "nkv": 8, "hd": 128, "rd": 128, "axes": 3,
         "interleaved": False, "block": 16, "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "layer", "experts", "experts", "mrope"])
    if op == "route":
        E = rng.choice([8, 60, 64, 128, 160, 256, 384])
        return {"op": op, "T": _log_int(rng, 1, 16384), "E": E, "k": rng.randint(1, min(8, E)), "shared": rng.random() < 0.5,
                "renorm": rng.random() < 0.7, "f32": rng.random() < 0.5, "masked": rng.random() < 0.4}
    if op == "mrope":
        hd = rng.choice([64, 128, 256])
        nkv = rng.choice([1, 2, 4, 8])
        return {"op": op, "T": _log_int(rng, 1, 12000), "nq": nkv * rng.choice([1, 4, 8]) if nkv < 8 else nkv * rng.choice([1, 4]),
                "nkv": nkv, "hd": hd, "rd": rng.choice([hd, hd // 2, hd // 4]), "axes": rng.choice([1, 2, 3]),
                "interleaved": rng.random() < 0.5, "block": rng.choice([16, 32, 64]), "pad": rng.choice([0, 0, 3])}
    while True:
        E = rng.choice([8, 16, 60, 64, 128, 256])
        k = rng.randint(1, min(8, E))
        H, I = 8 * _log_int(rng, 32, 512), 8 * _log_int(rng, 16, 512)
        T = _log_int(rng, 1, 200 if op == "layer" else 4096)
        if E * 3 * H * I * 2 <= 1.7e9 and 6.0 * T * k * H * I <= 4e11:
            break
    if op == "layer":
        return {"op": op, "T": T, "E": E, "k": k, "H": H, "I": I, "shared": rng.random() < 0.5}
    return {"op": op, "T": T, "E": E, "k": k, "H": H, "I": I, "pad": rng.choice([0, 0, 1, 5])}


# ----------------------------------------------------------------------------------------------------- inputs
def _logits(case, g, T, E):
    """Router logits of order one with some experts more popular than others."""
    cols = E + int(bool(case.get("shared")))
    l = torch.randn(T, cols, device="cuda", generator=g) + 0.3 * torch.randn(1, cols, device="cuda", generator=g)
    return l.to(torch.float32 if case.get("f32") else BF16)


def _weights(E, rows, cols, g, scale):
    return torch.empty(E, rows, cols, device="cuda", dtype=BF16).normal_(0.0, scale, generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, T = case["op"], case["T"]
    s = {"case": dict(case)}
    if op == "route":
        E = case["E"]
        l = _logits(case, g, T, E)
        if case["masked"]:
            off = torch.rand(T, E, device="cuda", generator=g) < 0.5
            off[-min(T, 3):] = True
            l[:, :E].masked_fill_(off, -math.inf)
        s["logits"] = l
        return s
    if op in ("layer", "experts"):
        E, k, H, I = case["E"], case["k"], case["H"], case["I"]
        n = E + int(bool(case.get("shared")))
        s["x"] = torch.randn(T, H, device="cuda", generator=g).to(BF16)
        s["w_gate_up"] = _weights(n, 2 * I, H, g, 1.0 / math.sqrt(H))
        s["w_down"] = _weights(n, H, I, g, 1.0 / math.sqrt(I))
        s["addend"] = torch.randn(T, H, device="cuda", generator=g).to(BF16)
        if op == "layer":
            s["logits"] = _logits(case, g, T, E)
            return s
        pick = torch.randn(T, E, device="cuda", generator=g) + 0.3 * torch.randn(1, E, device="cuda", generator=g)
        v, ids = pick.topk(k, dim=1)
        ids = ids.to(torch.int32)
        if case["pad"]:
            ids[-min(T, case["pad"]):] = -1
        s["ids"], s["weights"] = ids, torch.softmax(v, 1)
        return s
    nq, nkv, hd, rd, block = case["nq"], case["nkv"], case["hd"], case["rd"], case["block"]
    s["qkv"] = torch.randn(T, (nq + 2 * nkv) * hd, device="cuda", generator=g).to(BF16)
    # a run of text, then frames of a grid: time moves slowly, height and width inside a frame; the context is long
    A, t = case["axes"], torch.arange(T, device="cuda")
    start = int(torch.randint(0, 200000, (1,), device="cuda", generator=g))
    grid = torch.stack([t // 64, (t // 8) % 8, t % 8])[:A] + start
    s["positions"] = torch.where(t < T // 4, t + start, grid + T // 4).to(torch.int64).contiguous()
    half = rd // 2
    s["inv_freq"] = 1.0 / (1e7 ** (torch.arange(0, rd, 2, dtype=torch.float32, device="cuda") / rd))
    sec = [half - (A - 1) * (half // 4)] + [half // 4] * (A - 1)
    i = torch.arange(half, device="cuda")
    if case["interleaved"]:
        a = i % A
        s["axes"] = torch.where(i < A * torch.tensor(sec, device="cuda")[a], a, torch.zeros_like(a)).to(torch.int32)
    else:
        s["axes"] = torch.repeat_interleave(torch.arange(A, device="cuda"), torch.tensor(sec, device="cuda")).to(torch.int32)
    nb = -(-T // block) + 2
    kv = torch.zeros(nb, nkv, block, 2 * hd, device="cuda", dtype=BF16)
    s["kv"] = kv
    s["key_cache"], s["value_cache"] = kv.transpose(1, 2).split(hd, dim=-1)
    table = torch.randperm(nb, device="cuda", generator=g)
    slots = table[t // block] * block + t % block
    if case["pad"]:
        slots[-min(T, case["pad"]):] = -1
    s["slot_mapping"] = slots.to(torch.int64)
    s["q_out"] = torch.empty(T, nq * hd, device="cuda", dtype=BF16)
    return s


# ----------------------------------------------------------------------------------------------------- plain forms
def _plain_route(logits, E, k, shared, renorm):
    l = logits[:, :E].float()
    l = torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l).clamp(max=FLT_MAX)
    v, i = torch.sort(l, dim=1, descending=True, stable=True)
    top, ids = v[:, :k], i[:, :k].to(torch.int32)
    e = torch.where(torch.isinf(v), torch.zeros_like(v), torch.exp(v - v[:, :1]))
    z = (e[:, :k] if renorm else e).sum(1, keepdim=True)
    none = torch.isinf(top)
    w = torch.where(none, torch.zeros_like(top), e[:, :k] / z)
    ids = torch.where(none, torch.full_like(ids, -1), ids)
    if shared:
        w = torch.cat([w, torch.sigmoid(logits[:, E:].float())], 1)
        ids = torch.cat([ids, torch.full_like(ids[:, :1], E)], 1)
    return w.contiguous(), ids.contiguous()


def _swiglu(x, wgu, wd):
    g, u = (x @ wgu.transpose(-1, -2)).chunk(2, dim=-1)
    return (g * torch.sigmoid(g) * u) @ wd.transpose(-1, -2)


def _plain_experts(x, wgu, wd, weights, ids, addend, shared):
    """The routed products as one batched product over the experts, rows padded to the fullest expert; the shared expert,
    which every token takes, as one product of its own."""
    T, H = x.shape
    xf, out = x.float(), addend.float()
    if shared:
        out = out + weights[:, -1:] * _swiglu(xf, wgu[-1].float(), wd[-1].float())
        weights, ids, wgu, wd = weights[:, :-1], ids[:, :-1], wgu[:-1], wd[:-1]
    k = ids.shape[1]
    flat = ids.reshape(-1).long()
    if T * k <= 640 and T * k * wgu.shape[1] * H <= 1 << 30:  # few places: their experts' weights, gathered
        e = flat.clamp(min=0)
        y = _swiglu(xf.repeat_interleave(k, 0)[:, None], wgu[e].float(), wd[e].float())[:, 0]
    else:
        order = torch.argsort(torch.where(flat < 0, wgu.shape[0], flat), stable=True)
        live = order[: int((flat >= 0).sum())]
        e = flat[live]
        count = torch.bincount(e, minlength=wgu.shape[0])
        first = torch.cumsum(count, 0) - count
        at = torch.arange(live.numel(), device=x.device) - first[e]
        rows = torch.zeros(wgu.shape[0], int(count.max()), H, device=x.device)
        rows[e, at] = xf[live // k]
        y = torch.zeros(T * k, H, device=x.device)
        y[live] = _swiglu(rows, wgu.float(), wd.float())[e, at]
    w = torch.where(ids < 0, torch.zeros_like(weights), weights)
    out = out + (w[..., None] * y.view(T, k, H)).sum(1)
    return out.to(BF16)


def _plain_mrope(s, case):
    nq, nkv, hd, rd = case["nq"], case["nkv"], case["hd"], case["rd"]
    T = s["qkv"].shape[0]
    ang = s["positions"][s["axes"].long()].T.double() * s["inv_freq"].double()
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    x = s["qkv"].float().view(T, nq + 2 * nkv, hd)
    qk = torch.cat([x[:, :nq], x[:, nq:nq + nkv] * 0.75], 1)
    a, b = qk[..., : rd // 2], qk[..., rd // 2: rd]
    r = torch.cat([a * cos - b * sin, b * cos + a * sin, qk[..., rd:]], -1).to(BF16)
    s["q_out"].copy_(r[:, :nq].reshape(T, -1))
    block, ok = case["block"], s["slot_mapping"] >= 0
    slot = s["slot_mapping"][ok]
    s["key_cache"][slot // block, slot % block] = r[:, nq:][ok]
    s["value_cache"][slot // block, slot % block] = x[:, nq + nkv:][ok].to(BF16)
    return {"q": s["q_out"], "kv": s["kv"]}


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from multi_modal_parallelism_b200 import kernels as K

        if op == "route":
            w, ids = K.moe_route(s["logits"], case["k"], renormalize=case["renorm"], shared=case["shared"])
            return {"weights": w, "ids": ids}
        if op == "layer":
            return K.moe_layer(s["x"], s["logits"], s["w_gate_up"], s["w_down"], case["k"], shared=case["shared"],
                               addend=s["addend"])
        if op == "experts":
            return K.moe_experts(s["x"], s["w_gate_up"], s["w_down"], s["weights"], s["ids"], addend=s["addend"])
        K.qkv_mrope_kv_write(s["qkv"], case["nq"], case["nkv"], case["hd"], s["positions"], s["inv_freq"], s["axes"], 0.75,
                             s["q_out"], s["key_cache"], s["value_cache"], s["slot_mapping"])
        return {"q": s["q_out"], "kv": s["kv"]}
    if op == "route":
        w, ids = _plain_route(s["logits"], case["E"], case["k"], case["shared"], case["renorm"])
        return {"weights": w, "ids": ids}
    if op == "layer":
        w, ids = _plain_route(s["logits"], case["E"], case["k"], case["shared"], True)
        return _plain_experts(s["x"], s["w_gate_up"], s["w_down"], w, ids, s["addend"], case["shared"])
    if op == "experts":
        return _plain_experts(s["x"], s["w_gate_up"], s["w_down"], s["weights"], s["ids"], s["addend"], False)
    return _plain_mrope(s, case)


# ----------------------------------------------------------------------------------------------------- floors
def work(case):
    op, T = case["op"], case["T"]
    if op == "route":
        n = case["E"] + int(case["shared"])
        return {"bytes": T * n * (4 if case["f32"] else 2) + T * (case["k"] + int(case["shared"])) * 8, "flops": 4 * T * n}
    if op == "mrope":
        row = (case["nq"] + 2 * case["nkv"]) * case["hd"]
        return {"bytes": T * (2 * row * 2 + 8 * case["axes"] + 8), "flops": 6 * T * (case["nq"] + case["nkv"]) * case["rd"] // 2}
    E, k, H, I = case["E"], case["k"], case["H"], case["I"]
    sh = int(bool(case.get("shared")))
    live = T - min(T, case.get("pad", 0))
    hit = E * (1.0 - (1.0 - k / E) ** live) + sh  # experts that at least one token takes, at even popularity
    b = hit * 3 * H * I * 2 + T * H * 2 * 3 + T * (k + sh) * 8
    if op == "layer":
        b += T * (E + sh) * 2 - T * (k + sh) * 8
    return {"bytes": int(b), "flops": 6 * live * (k + sh) * H * I}


# ----------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    def route(logits, renorm):
        E, k = case["E"], case["k"]
        l = logits.double()
        w = torch.zeros(l.shape[0], k + int(case["shared"]), dtype=torch.float64, device=l.device)
        ids = torch.full(w.shape, -1, dtype=torch.int32, device=l.device)
        left = l[:, :E].clone()
        p = torch.softmax(left.masked_fill((left == -math.inf).all(1, keepdim=True), 0.0), 1)
        for j in range(k):
            best = left.max(1).values
            at = (left == best[:, None]).to(torch.int8).argmax(1)
            ok = best > -math.inf
            ids[:, j] = torch.where(ok, at, -1).to(torch.int32)
            w[:, j] = torch.where(ok, p.gather(1, at[:, None])[:, 0], 0.0)
            left.scatter_(1, at[:, None], -math.inf)
        if renorm:
            z = w[:, :k].sum(1, keepdim=True)
            w[:, :k] = torch.where(z > 0, w[:, :k] / z, 0.0)
        if case["shared"]:
            w[:, k] = 1.0 / (1.0 + torch.exp(-l[:, E]))
            ids[:, k] = E
        return w, ids

    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        w, ids = route(s["logits"], case["renorm"])
        return {"weights": w, "ids": None}
    if op == "mrope":
        nq, nkv, hd, h = case["nq"], case["nkv"], case["hd"], case["rd"] // 2
        T = case["T"]
        x = s["qkv"].double().view(T, nq + 2 * nkv, hd)
        q, k, v = x[:, :nq].clone(), 0.75 * x[:, nq:nq + nkv], x[:, nq + nkv:]
        for i in range(h):
            a = s["positions"][int(s["axes"][i])].double() * float(s["inv_freq"][i])
            z = torch.complex(a.cos(), a.sin())[:, None]
            for t in (q, k):
                r = torch.complex(t[..., i], t[..., i + h]) * z
                t[..., i], t[..., i + h] = r.real.clone(), r.imag.clone()
        kv = torch.zeros(s["kv"].shape, dtype=torch.float64, device="cuda")
        ok = s["slot_mapping"] >= 0
        slot = s["slot_mapping"][ok]
        kv[slot // case["block"], :, slot % case["block"]] = torch.cat([k, v], -1)[ok]
        return {"q": q.reshape(T, -1), "kv": kv}
    E, k, T = case["E"], case["k"], case["T"]
    if op == "layer":
        w, ids = route(s["logits"], True)
    else:
        w, ids = s["weights"].double(), s["ids"]
    x, out = s["x"].double(), s["addend"].double()
    for e in range(s["w_down"].shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel():
            gu = s["w_gate_up"][e].double() @ x[t].T
            g, u = gu[: case["I"]], gu[case["I"]:]
            out.index_add_(0, t, w[t, j][:, None] * (s["w_down"][e].double() @ (g / (1.0 + torch.exp(-g)) * u)).T)
    return out
