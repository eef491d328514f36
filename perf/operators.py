"""What is measured of three operators, and their plain forms.

linear  y = act((xq . w) * xs * ws + bias) + residual: the W8A8 product of the linear layers
        with its epilogue (``ops.linear_w8a8``).
chunk   attention of a chunk of new tokens per sequence over the paged int8 K/V cache, causal
        at the end of each sequence's context (``ops.paged_chunk_q8``).
moe     a whole sparse-MoE feed-forward for a few tokens: router, top-k, the chosen experts'
        W8A8 gate_up, SwiGLU and down products, weighted sum (``ops.moe_layer``).

Sizes are those of this repository's configurations (8B: hidden 4096, 32/8 heads, FFN 12288;
27B: 40/8 heads; 30B-A3B: hidden 2048, 32/4 heads, 128 experts top-8 of 768) and odd ones
between them. Head dimension is 128 throughout, as everywhere in the framework.
"""

import math
import random

import torch

own = False

HD = 128
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _dev():
    return "cuda" if torch.cuda.is_available() else "cpu"


# ------------------------------------------------------------------------------- cases ----
def listed():
    return [
        # the output projection and its residual for eight decoding rows: one read of the weights
        {"name": "linear_rows8", "op": "linear", "M": 8, "N": 4096, "K": 4096, "dtype": "bf16",
         "act": "none", "bias": False, "residual": True},
        # nothing a multiple of a tile: a projector's first layer over an image's patches
        {"name": "linear_ragged", "op": "linear", "M": 999, "N": 5127, "K": 1040, "dtype": "fp16",
         "act": "gelu", "bias": True, "residual": False},
        # the output projection of a 4096-token prompt chunk, with bias and residual
        {"name": "linear_chunk4096", "op": "linear", "M": 4096, "N": 4096, "K": 4096,
         "dtype": "bf16", "act": "none", "bias": True, "residual": True},
        # the gate projection of eight 1024-token prompts, SiLU applied on the way out
        {"name": "linear_chunk8192", "op": "linear", "M": 8192, "N": 12288, "K": 4096,
         "dtype": "bf16", "act": "silu", "bias": False, "residual": False},
        # the first tokens of a small model's only request: latency alone
        {"name": "chunk_tiny", "op": "chunk", "S": 1, "n": 5, "ctx": 37, "Hq": 4, "Hkv": 2,
         "bs": 16, "dtype": "bf16"},
        # four draft tokens of each of 64 running sequences are checked at once
        {"name": "chunk_verify", "op": "chunk", "S": 64, "n": 4, "ctx": 2048, "Hq": 32, "Hkv": 8,
         "bs": 16, "dtype": "bf16"},
        # a short question after a long document: few rows, a long cache
        {"name": "chunk_long_cache", "op": "chunk", "S": 2, "n": 16, "ctx": 65536, "Hq": 40,
         "Hkv": 8, "bs": 16, "dtype": "bf16"},
        # eight prompts of up to 2048 tokens, from the first token on
        {"name": "chunk_prompts", "op": "chunk", "S": 8, "n": 2048, "ctx": 2048, "Hq": 32,
         "Hkv": 8, "bs": 16, "dtype": "bf16"},
        # the last quarter of a 16K prompt, in one chunk
        {"name": "chunk_late", "op": "chunk", "S": 1, "n": 4096, "ctx": 16384, "Hq": 32,
         "Hkv": 4, "bs": 64, "dtype": "fp16"},
        # one decoding row: the least there is to do
        {"name": "moe_one", "op": "moe", "T": 1, "H": 2048, "F": 768, "E": 128, "k": 8,
         "dtype": "bf16", "norm": True},
        # eight decoding rows: most of their experts have one row each
        {"name": "moe_eight", "op": "moe", "T": 8, "H": 2048, "F": 768, "E": 128, "k": 8,
         "dtype": "bf16", "norm": True},
        # sixteen rows over few experts of odd sizes: several rows to an expert
        {"name": "moe_ragged16", "op": "moe", "T": 16, "H": 1040, "F": 272, "E": 20, "k": 3,
         "dtype": "fp16", "norm": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "chunk", "moe"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "linear":
        while True:
            M, N, K = _log(rng, 1, 8192), _log(rng, 16, 24576), 16 * _log(rng, 4, 768)
            if M * N * K <= 8192 * 12288 * 4096:
                break
        return {"op": op, "M": M, "N": N, "K": K, "dtype": dtype,
                "act": rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    if op == "chunk":
        Hq, Hkv = rng.choice([(4, 2), (16, 8), (32, 8), (40, 8), (32, 4), (8, 8), (21, 3), (24, 2)])
        while True:
            S, n, ctx = _log(rng, 1, 64), _log(rng, 1, 4096), _log(rng, 16, 65536)
            if n <= ctx and S * ctx <= 131072 and S * Hq * n * ctx <= 4096 * 16384 * 32:
                break
        return {"op": op, "S": S, "n": n, "ctx": ctx, "Hq": Hq, "Hkv": Hkv,
                "bs": rng.choice([4, 8, 16, 16, 32, 64, 256]), "dtype": dtype}
    E = rng.choice([8, 16, 20, 64, 128])
    return {"op": op, "T": rng.randint(1, 16), "H": 16 * rng.randint(16, 160),
            "F": 16 * rng.randint(8, 80), "E": E, "k": rng.randint(1, min(8, E)),
            "dtype": dtype, "norm": rng.random() < 0.7}


def _lens(case):
    """(new tokens, context) of every sequence: the first is the longest, the others ragged; a
    sequence in eight or so brings no new token."""
    r = random.Random("%(S)d %(n)d %(ctx)d %(Hq)d %(bs)d" % case)
    out = [(case["n"], case["ctx"])]
    for _ in range(case["S"] - 1):
        n = 0 if r.random() < 0.12 else r.randint(max(1, case["n"] // 2), case["n"])
        c = n if case["n"] == case["ctx"] else r.randint(max(n, case["ctx"] // 2), case["ctx"])
        out.append((n, max(c, n)))
    return out


def _pairs(case):
    return sum(n * (c - n) + n * (n + 1) // 2 for n, c in _lens(case))


def work(case):
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        b = M * K + N * K + 4 * (M + N) + 2 * M * N * (2 if case["residual"] else 1)
        return {"bytes": b + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    if case["op"] == "chunk":
        lens = _lens(case)
        T = sum(n for n, _ in lens)
        keys = sum(c for n, c in lens if n)
        b = keys * case["Hkv"] * 2 * (HD + 4) + T * case["Hq"] * (HD + 4 + 2 * HD)
        return {"bytes": b + 4 * keys // case["bs"], "flops": 4 * HD * case["Hq"] * _pairs(case)}
    T, H, F, E, k = (case[x] for x in ("T", "H", "F", "E", "k"))
    hit = E * (1 - (1 - k / E) ** T)  # experts that some row chose, on average
    return {"bytes": hit * (3 * H * F + 8 * F + 4 * H) + 4 * E * H + T * H * 5,
            "flops": 2 * T * k * 3 * H * F + 2 * T * E * H}


# ------------------------------------------------------------------------------ inputs ----
def _gen(seed):
    g = torch.Generator(device=_dev())
    g.manual_seed(seed)
    return g


def _codes(g, *shape):
    """int8 codes of rows of normal values whose largest is about 3.5 deviations."""
    return (36.3 * torch.randn(shape, generator=g, device=_dev())).round().clamp(-127, 127).to(torch.int8)


def _uniform(g, lo, hi, *shape):
    return lo + (hi - lo) * torch.rand(shape, generator=g, device=_dev())


def _quant(x):
    """Per-row int8 codes and scales of dtype rows, as the norm before these layers gives."""
    a = x.float().abs().amax(-1, keepdim=True)
    q = torch.round(x.float() * (127.0 / a)).clamp(-127, 127).to(torch.int8)
    return q, (a / 127.0).squeeze(-1)


def prepare(case, seed):
    g, dt, dev = _gen(seed), DT[case["dtype"]], _dev()
    s = {"case": dict(case)}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["xq"], s["xs"] = _codes(g, M, K), _uniform(g, 0.01, 0.04, M)
        s["w"], s["ws"] = _codes(g, N, K), _uniform(g, 0.5, 1.5, N) / (36.3 * math.sqrt(K))
        s["bias"] = torch.randn(N, generator=g, device=dev).to(dt) if case["bias"] else None
        s["res"] = torch.randn(M, N, generator=g, device=dev).to(dt) if case["residual"] else None
        if own:
            from superl8_serve_b200 import ops

            s["space"] = ops.linear_workspace(M, N, K, dev)
    elif case["op"] == "chunk":
        Hq, Hkv, bs = case["Hq"], case["Hkv"], case["bs"]
        lens = _lens(case)
        T, S = sum(n for n, _ in lens), len(lens)
        need = [-(-c // bs) for _, c in lens]
        nb = sum(need) + 3
        perm = torch.randperm(nb, generator=g, device=dev).to(torch.int32)
        at = torch.tensor([sum(need[:i]) for i in range(S)], device=dev)
        col = torch.arange(max(need), device=dev)
        idx = (at[:, None] + col).clamp(max=nb - 1)
        fits = col < torch.tensor(need, device=dev)[:, None]
        s["bt"] = torch.where(fits, perm[idx], torch.zeros_like(perm[idx])).contiguous()
        s["kc"], s["vc"] = _codes(g, nb, Hkv, bs, HD), _codes(g, nb, Hkv, bs, HD)
        s["ks"] = _uniform(g, 0.02, 0.04, nb, Hkv, bs)
        s["vs"] = _uniform(g, 0.01, 0.05, nb, Hkv, bs)
        s["q"], s["qs"] = _codes(g, T, Hq, HD), _uniform(g, 0.02, 0.08, T, Hq)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        s["ctx"] = i32([c for _, c in lens])
        s["cu"] = i32([sum(n for n, _ in lens[:i]) for i in range(S + 1)])
        # where each new token stands: its sequence and its place among the sequence's new ones
        s["seq"] = torch.tensor([i for i, (n, _) in enumerate(lens) for _ in range(n)], device=dev)
        s["at"] = torch.tensor([j for n, _ in lens for j in range(n)], device=dev)
        s["longest"] = (max(n for n, _ in lens), max(c for _, c in lens))
        s["scale"] = HD ** -0.5
        if own:
            from superl8_serve_b200 import ops

            s["space"] = ops.chunk_workspace(dev)
    else:
        T, H, F, E = case["T"], case["H"], case["F"], case["E"]
        s["y"] = torch.randn(T, H, generator=g, device=dev).to(dt)
        s["xq"], s["xs"] = _quant(s["y"])
        s["gate"] = 0.02 * math.sqrt(2048 / H) * torch.randn(E, H, generator=g, device=dev)
        s["gu_w"], s["d_w"] = _codes(g, E, 2 * F, H), _codes(g, E, H, F)
        s["gu_s"] = _uniform(g, 0.5, 1.5, E, 2 * F) / (36.3 * math.sqrt(H))
        s["d_s"] = _uniform(g, 0.5, 1.5, E, H) / (36.3 * math.sqrt(F))
        if own:
            from superl8_serve_b200 import ops

            s["space"] = ops.moe_layer_workspace(case["k"], F, dev)
    return s


# --------------------------------------------------------------------------- the passes ----
def _act(v, name):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v.clamp(min=0) if name == "relu" else v


def _plain_linear(s):
    c, dt = s["case"], DT[s["case"]["dtype"]]
    v = (s["xq"].float() @ s["w"].float().T) * s["xs"][:, None] * s["ws"]
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _act(v, c["act"])
    if s["res"] is not None:
        v = v + s["res"].float()
    return v.to(dt)


def _plain_chunk(s):
    c = s["case"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    G, S = Hq // Hkv, s["ctx"].shape[0]
    nmax, cmax = s["longest"]
    T = s["q"].shape[0]
    bt = s["bt"].long()
    k = (s["kc"][bt].float() * s["ks"][bt][..., None]).transpose(1, 2).reshape(S, Hkv, -1, HD)
    v = (s["vc"][bt].float() * s["vs"][bt][..., None]).transpose(1, 2).reshape(S, Hkv, -1, HD)
    q = torch.zeros(S, nmax, Hkv, G, HD, device=k.device)
    q[s["seq"], s["at"]] = (s["q"].float() * s["qs"][..., None]).reshape(T, Hkv, G, HD)
    q = q.permute(0, 2, 1, 3, 4).reshape(S, Hkv, nmax * G, HD)
    x = (q @ k[:, :, :cmax].transpose(-1, -2)).mul_(s["scale"])
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    last = s["ctx"].long()[:, None] - new[:, None] + torch.arange(nmax, device=k.device)
    last = last.repeat_interleave(G, 1)  # the last position that each row sees
    hide = torch.arange(cmax, device=k.device) > last[..., None]
    x.masked_fill_(hide[:, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    den = x.sum(-1, keepdim=True)
    o = (x @ v[:, :, :cmax]) / torch.where(den == 0, 1.0, den)
    o = o.reshape(S, Hkv, nmax, G, HD).permute(0, 2, 1, 3, 4)[s["seq"], s["at"]]
    return o.reshape(T, Hq * HD).to(DT[c["dtype"]])


def _plain_moe(s):
    c = s["case"]
    F, k = c["F"], c["k"]
    # the choice of experts hangs on values that lie close together: in 64 bits
    p = (s["y"].double() @ s["gate"].double().T)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    order = torch.sort(p, dim=-1, descending=True, stable=True)
    w, e = order.values[:, :k].float(), order.indices[:, :k]
    if c["norm"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-9)
    gu = torch.einsum("th,tkfh->tkf", s["xq"].float(), s["gu_w"][e].float())
    gu = gu * s["xs"][:, None, None] * s["gu_s"][e]
    a = _act(gu[..., :F], "silu") * gu[..., F:]
    top = a.abs().amax(-1, keepdim=True)
    aq = torch.round(a * torch.where(top > 0, 127.0 / top, 0.0)).clamp(-127, 127)
    d = torch.einsum("tkf,tkhf->tkh", aq, s["d_w"][e].float())
    d = d * (top / 127.0) * s["d_s"][e]
    return (d * w[..., None]).sum(1).to(DT[c["dtype"]])


def run(state):
    s, c = state, state["case"]
    if own:
        from superl8_serve_b200 import ops

        if c["op"] == "linear":
            return ops.linear_w8a8(s["xq"], s["xs"], s["w"], s["ws"], bias=s["bias"],
                                   activation=None if c["act"] == "none" else c["act"],
                                   residual=s["res"], out_dtype=DT[c["dtype"]],
                                   workspace=s["space"])
        if c["op"] == "chunk":
            return ops.paged_chunk_q8(s["q"], s["qs"], s["kc"], s["ks"], s["vc"], s["vs"], s["bt"],
                                      s["ctx"], s["cu"], s["scale"], workspace=s["space"],
                                      dtype=DT[c["dtype"]])
        return ops.moe_layer(s["y"], s["xq"], s["xs"], s["gate"], s["gu_w"], s["gu_s"], s["d_w"],
                             s["d_s"], c["k"], norm_topk_prob=c["norm"], workspace=s["space"])
    return {"linear": _plain_linear, "chunk": _plain_chunk, "moe": _plain_moe}[c["op"]](s)


# --------------------------------------------------------------------------- in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "linear":
        y = torch.empty(case["M"], case["N"], dtype=f64, device=_dev())
        w = s["w"].to(f64)
        for i in range(0, case["M"], 1024):
            r = slice(i, i + 1024)
            z = torch.matmul(s["xq"][r].to(f64), w.t())
            z = z.mul(s["xs"][r].to(f64).unsqueeze(1)).mul(s["ws"].to(f64))
            if s["bias"] is not None:
                z = z + s["bias"].to(f64)
            if case["act"] == "silu":
                z = z * torch.sigmoid(z)
            elif case["act"] == "gelu":
                z = torch.special.ndtr(z) * z
            elif case["act"] == "gelu_tanh":
                z = z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * z * (1 + 0.044715 * z ** 2))
            elif case["act"] == "relu":
                z = torch.where(z > 0, z, torch.zeros_like(z))
            y[r] = z if s["res"] is None else z + s["res"][r].to(f64)
        return y
    if case["op"] == "chunk":
        Hq, Hkv, bs = case["Hq"], case["Hkv"], case["bs"]
        y = torch.zeros(s["q"].shape[0], Hq, HD, dtype=f64, device=_dev())
        row = 0
        for i, (n, c) in enumerate(_lens(case)):
            if n == 0:
                continue
            pos = torch.arange(c, device=_dev())
            blk, off = s["bt"][i].long()[pos // bs], pos % bs
            seen = pos <= c - n + torch.arange(n, device=_dev()).unsqueeze(1)
            for h in range(Hq):
                j = h * Hkv // Hq
                k = s["kc"][blk, j, off].to(f64) * s["ks"][blk, j, off].to(f64).unsqueeze(1)
                v = s["vc"][blk, j, off].to(f64) * s["vs"][blk, j, off].to(f64).unsqueeze(1)
                q = s["q"][row:row + n, h].to(f64) * s["qs"][row:row + n, h].to(f64).unsqueeze(1)
                z = torch.einsum("rd,pd->rp", q, k) * s["scale"]
                z[~seen] = float("-inf")
                y[row:row + n, h] = torch.softmax(z, -1) @ v
            row += n
        return y.reshape(-1, Hq * HD)
    T, F, k = case["T"], case["F"], case["k"]
    y = torch.zeros(T, case["H"], dtype=f64, device=_dev())
    prob = torch.softmax(torch.einsum("th,eh->te", s["y"].to(f64), s["gate"].to(f64)), -1)
    for t in range(T):
        chosen = sorted(range(case["E"]), key=lambda e: (-float(prob[t, e]), e))[:k]
        total = max(float(prob[t, chosen].sum()), 1e-9) if case["norm"] else 1.0
        for e in chosen:
            x = torch.mv(s["gu_w"][e].to(f64), s["xq"][t].to(f64)) * float(s["xs"][t]) * s["gu_s"][e].to(f64)
            a = x[:F] * torch.sigmoid(x[:F]) * x[F:]
            step = a.abs().max() / 127
            code = torch.round(a / step) if float(step) > 0 else torch.zeros_like(a)
            y[t] += float(prob[t, e]) / total * step * s["d_s"][e].to(f64) * torch.mv(s["d_w"][e].to(f64), code)
    return y
