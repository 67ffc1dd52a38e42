"""The calls that tune a router and low-rank adapters on top of frozen experts,
and that serve many adapters at once: their inputs, their plain forms, their
work and a float64 restatement of their results.

Five operators, reached through ffai_amd.tuning:

  balance_loss        per-expert counts, probability sums, balance and z loss
  router_backward     gradient of the router's logits
  unpermute_backward  gradient of the weighted combine
  LoRAAdapters.apply      y + scale * B (A x), an adapter for each row
  LoRAAdapters.backward   its gradients with respect to x, A and B

Where `own` is false `run` computes them from elementary torch operations in
32 bits, otherwise through the library.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# Fields of a case by operator:
#   balance / router:  T rows, E experts, k picks, gating ("softmax_topk",
#     "topk_softmax", "sigmoid"), norm (renormalised weights), eb (an expert
#     bias that shifts the selection), pad (share of rows that are padding),
#     skew (spread of the experts' popularity)
#   combine:  T rows, k picks, E experts, H hidden
#   lora / lora_bwd:  T rows, K inputs, N outputs, R rank, G adapters, reqs
#     (requests the rows belong to; 0: one per row), none (share of the
#     requests without an adapter)
ROUTER = dict(gating="softmax_topk", norm=True, eb=False, pad=0.0, skew=0.5, dt="bf16")
LORA = dict(reqs=0, none=0.0, dt="bf16")


def listed():
    return [
        # a small batch on a layer of few large experts: launches and host work
        dict(ROUTER, name="balance_t64_e32", op="balance", T=64, E=32, k=4, gating="topk_softmax"),
        # eight sequences of 4096 tokens, padded at their ends, on 256 small experts
        dict(ROUTER, name="balance_t32768_e256", op="balance", T=32768, E=256, k=8, pad=0.1, skew=1.0),
        # one odd-length sequence through a sigmoid router with a selection bias, f16
        dict(ROUTER, name="router_bwd_t333_e128", op="router", T=333, E=128, k=6, gating="sigmoid", eb=True, dt="f16"),
        # a large training batch on 128 experts
        dict(ROUTER, name="router_bwd_t32768_e128", op="router", T=32768, E=128, k=8, pad=0.05, skew=1.0),
        # a short odd batch on few large experts
        dict(name="combine_bwd_t37_h2880", op="combine", T=37, E=32, k=4, H=2880, dt="bf16"),
        # a training sequence on 128 experts
        dict(name="combine_bwd_t4096_h2048", op="combine", T=4096, E=128, k=8, H=2048, dt="bf16"),
        # one token of one request, the adapter of a small up projection
        dict(LORA, name="lora_t1_r16", op="lora", T=1, K=2048, N=768, R=16, G=64),
        # a decode batch of 64 requests, each with its own adapter or none
        dict(LORA, name="lora_t64_r16", op="lora", T=64, K=2048, N=2048, R=16, G=64, none=0.1),
        # ragged prompts of a few requests, f16, a rank between the usual ones, wide rows
        dict(LORA, name="lora_t1000_r24", op="lora", T=1000, K=2880, N=2880, R=24, G=32, reqs=5, none=0.2, dt="f16"),
        # long prompts, high rank
        dict(LORA, name="lora_t4096_r64", op="lora", T=4096, K=2048, N=2048, R=64, G=16, reqs=8),
        # tuning one small adapter on one odd-length sequence, f32
        dict(LORA, name="lora_bwd_t333_r8", op="lora_bwd", T=333, K=1024, N=384, R=8, G=1, reqs=1, dt="f32"),
        # tuning eight adapters at once on a batch of 4096 tokens
        dict(LORA, name="lora_bwd_t4096_r16", op="lora_bwd", T=4096, K=2048, N=2048, R=16, G=8, reqs=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    while True:
        op = rng.choice(["balance", "router", "combine", "lora", "lora", "lora_bwd"])
        dt = rng.choice(["bf16", "bf16", "f16", "f32"])
        if op in ("balance", "router"):
            E = rng.choice([8, 16, 32, 60, 64, 96, 128, 160, 256, rng.randint(5, 512)])
            c = dict(op=op, T=_log(rng, 1, 65536), E=E, k=rng.randint(1, min(E, rng.choice([2, 8, 8, 16]))),
                     gating=rng.choice(["softmax_topk", "softmax_topk", "topk_softmax", "sigmoid"]),
                     norm=rng.random() < 0.7, eb=rng.random() < 0.3, pad=rng.choice([0.0, 0.0, 0.1, 0.5]),
                     skew=rng.choice([0.0, 0.5, 1.5]), dt=dt)
        elif op == "combine":
            E = rng.choice([8, 32, 60, 128, 256])
            c = dict(op=op, T=_log(rng, 1, 8192), E=E, k=rng.randint(1, min(E, 10)), H=8 * _log(rng, 8, 512), dt=dt)
        else:
            T = _log(rng, 1, 8192)
            G = _log(rng, 1, 64)
            reqs = 0 if op == "lora" and T <= 256 and rng.random() < 0.7 else min(T, _log(rng, 1, 64))
            c = dict(op=op, T=T, K=8 * _log(rng, 8, 512), N=8 * _log(rng, 8, 512),
                     R=rng.choice([8, 16, 16, 24, 32, 40, 64, 128]), G=G, reqs=reqs,
                     none=rng.choice([0.0, 0.0, 0.2]), dt=dt)
        w = work(c)
        if w["flops"] <= 2.2e9 and w["bytes"] <= 290e6:
            return c


def work(case):
    c = case
    es = 4 if c["dt"] == "f32" else 2
    if c["op"] == "balance":  # logits, ids, mask in; counts, sums and losses out
        return {"bytes": c["T"] * (c["E"] * es + 4 * c["k"] + 1) + 8 * c["E"] + 12,
                "flops": 5 * c["T"] * c["E"]}
    if c["op"] == "router":  # logits, ids, gradients of the weights, mask in; gradient of the logits out
        return {"bytes": c["T"] * (2 * c["E"] * es + 8 * c["k"] + 1) + 4 * c["E"],
                "flops": 10 * c["T"] * c["E"]}
    if c["op"] == "combine":  # gradient of the output, expert rows in; gradients of the rows and the weights out
        M = c["T"] * c["k"]
        return {"bytes": es * c["H"] * (c["T"] + 2 * M) + 12 * M, "flops": 3 * M * c["H"]}
    used = min(c["G"], c["T"] if c["reqs"] == 0 else c["reqs"])
    T, K, N, R = c["T"], c["K"], c["N"], c["R"]
    ab = R * (K + N) * es
    if c["op"] == "lora":  # x and the rows to add to in, adapters in; rows out
        return {"bytes": T * (K + 2 * N) * es + used * ab + 4 * T, "flops": 2 * T * R * (K + N)}
    # x, dy and dx in, adapters in; dx and the adapters' gradients out
    return {"bytes": T * (3 * K + N) * es + used * ab + c["G"] * ab + 4 * T, "flops": 6 * T * R * (K + N)}


# ---------------------------------------------------------------- inputs --

def _randn(gen, *shape, std=1.0):
    return torch.randn(*shape, device="cuda", generator=gen).mul_(std)


def _routing(c, gen):
    """Logits as a router leaves them, the picks of its rule, padding rows."""
    T, E, k, dt = c["T"], c["E"], c["k"], DTYPES[c["dt"]]
    pop = _randn(gen, E, std=c["skew"])
    logits = _randn(gen, T, E).add_(pop).to(dt)
    eb = None
    if c["eb"] and c["gating"] != "topk_softmax":
        top = 0.05 if c["gating"] == "sigmoid" else 0.5 / E
        eb = torch.empty(E, device="cuda").uniform_(0.0, top, generator=gen)
    score = logits.float()
    if c["gating"] == "sigmoid":
        score = torch.sigmoid(score)
    elif c["gating"] == "softmax_topk" and eb is not None:
        score = torch.softmax(score, -1)
    if eb is not None:
        score = score + eb
    idx = torch.topk(score, k, dim=-1).indices.to(torch.int32).contiguous()
    mask = None
    if c["pad"] > 0:
        mask = torch.rand(T, device="cuda", generator=gen) >= c["pad"]
    return logits, idx, mask, eb


def _requests(c, gen):
    """The adapter of each row: rows belong to requests of ragged lengths."""
    T, G = c["T"], c["G"]
    n = c["reqs"] or T
    ad = torch.randint(0, G, (n,), device="cuda", generator=gen)
    if c["none"] > 0:
        ad = torch.where(torch.rand(n, device="cuda", generator=gen) < c["none"], torch.full_like(ad, -1), ad)
    if c["reqs"]:
        cuts = torch.rand(T, device="cuda", generator=gen).argsort()[: n - 1]
        step = torch.zeros(T, dtype=torch.int64, device="cuda")
        step[cuts] = 1
        ad = ad[step.cumsum(0).clamp_(max=n - 1)]
    return ad.to(torch.int32).contiguous()


def _scales(c):
    """The scales of a router: (of its logits, of its weights)."""
    return 1.0, 2.5 if c["gating"] == "sigmoid" else 1.0


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dt"]]
    s = dict(case=c)
    if c["op"] in ("balance", "router"):
        s["logits"], s["idx"], s["mask"], s["eb"] = _routing(c, gen)
        if c["op"] == "router":
            valid = torch.ones(c["T"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
            picks = s["idx"][valid].flatten().long()
            counts = torch.zeros(c["E"] + 1, dtype=torch.int32, device="cuda")
            counts[:-1] = torch.bincount(picks, minlength=c["E"]).int()
            counts[-1] = valid.sum().int()
            s["counts"] = counts
            s["dw"] = _randn(gen, c["T"], c["k"], std=0.05)
            s["coefs"] = (0.01, 0.001)
        if own:
            s["router"] = _router(c, s["eb"])
    elif c["op"] == "combine":
        T, E, k, H = c["T"], c["E"], c["k"], c["H"]
        idx = torch.rand(T, E, device="cuda", generator=gen).topk(k).indices
        perm = idx.flatten().argsort(stable=True)
        inv = torch.empty_like(perm)
        inv[perm] = torch.arange(T * k, device="cuda")
        s["inv"] = inv.to(torch.int32).reshape(T, k)
        s["w"] = torch.softmax(_randn(gen, T, k), -1)
        s["Y"] = _randn(gen, T * k, H).to(dt)
        s["dout"] = _randn(gen, T, H, std=0.02).to(dt)
    else:
        T, K, N, R, G = c["T"], c["K"], c["N"], c["R"], c["G"]
        s["x"] = _randn(gen, T, K).to(dt)
        s["A"] = _randn(gen, G, R, K, std=K ** -0.5).to(dt)
        s["B"] = _randn(gen, G, N, R, std=0.05).to(dt)
        s["scale"] = torch.empty(G, device="cuda").uniform_(0.5, 2.0, generator=gen)
        s["ad"] = _requests(c, gen)
        if c["op"] == "lora":
            s["y"] = _randn(gen, T, N).to(dt)
            s["out"] = torch.empty_like(s["y"])
        else:
            s["dy"] = _randn(gen, T, N, std=0.02).to(dt)
            s["dx"] = _randn(gen, T, K, std=0.02).to(dt)
            s["dx_out"] = torch.empty_like(s["dx"])
        if own:
            from ffai_amd.tuning import LoRAAdapters
            s["lora"] = LoRAAdapters(s["A"], s["B"], s["scale"])
    return s


def _router(c, eb):
    from ffai_amd.layer import MoEGatingMode, MoERouter
    mode = {"softmax_topk": MoEGatingMode.softmaxThenTopK, "topk_softmax": MoEGatingMode.topKThenSoftmax,
            "sigmoid": MoEGatingMode.sigmoidTopK}[c["gating"]]
    ls, rs = _scales(c)
    return MoERouter(c["E"], c["k"], mode, c["norm"], eb, ls, rs)


# ------------------------------------------------------------------- run --

def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from ffai_amd import tuning
    op = s["case"]["op"]
    if op == "balance":
        b = tuning.balance_loss(s["router"], s["logits"], s["idx"], mask=s["mask"])
        return {"counts": b.counts, "prob_sum": b.prob_sum, "losses": b.losses}
    if op == "router":
        return tuning.router_backward(s["router"], s["logits"], s["idx"], d_weight=s["dw"], counts=s["counts"],
                                      balance_coef=s["coefs"][0], z_coef=s["coefs"][1], mask=s["mask"])
    if op == "combine":
        return tuning.unpermute_backward(s["dout"], s["Y"], s["inv"], s["w"])
    if op == "lora":
        return s["lora"].apply(s["x"], s["ad"], s["y"], out=s["out"])
    return s["lora"].backward(s["x"], s["dy"], s["ad"], dx=s["dx"], dx_out=s["dx_out"])


def _probs(c, s):
    """The router's probabilities over all experts, for the losses."""
    if c["gating"] == "sigmoid":
        q = 1.0 / (1.0 + torch.exp(-s))
        return q / q.sum(-1, keepdim=True)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _lse(s):
    m = s.amax(-1)
    return m + torch.log(torch.exp(s - m[:, None]).sum(-1))


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "balance":
        return _plain_balance(c, s)
    if op == "router":
        return _plain_router(c, s)
    if op == "combine":
        dt = s["Y"].dtype
        inv = s["inv"].long()
        g, Y = s["dout"].float(), s["Y"].float()
        w = s["w"].to(dt).float()
        dw = (g[:, None, :] * Y[inv]).sum(-1)
        dY = torch.empty_like(s["Y"])
        dY[inv.flatten()] = (w[:, :, None] * g[:, None, :]).to(dt).reshape(-1, c["H"])
        return dY, dw
    # the adapters side by side: A as [G R, K], B as [N, G R]; a row keeps the
    # part of its own adapter
    G, R, K, N = c["G"], c["R"], c["K"], c["N"]
    dt = s["x"].dtype
    x, ad = s["x"].float(), s["ad"].long()
    A = s["A"].float().reshape(G * R, K)
    B = s["B"].float().permute(0, 2, 1).reshape(G * R, N)
    keep = (ad[:, None] == torch.arange(G, device=ad.device)).float() * s["scale"]
    keep = keep[:, :, None].expand(-1, G, R).reshape(-1, G * R)
    xa = (x @ A.t()) * keep
    if op == "lora":
        return (s["y"].float() + xa @ B).to(dt)
    dy = s["dy"].float()
    u = (dy @ B.t()) * keep
    dx = (s["dx"].float() + u @ A).to(dt)
    dA = (u.t() @ x).reshape(G, R, K).to(dt)
    dB = (dy.t() @ xa).reshape(N, G, R).permute(1, 0, 2).contiguous().to(dt)
    return dx, dA, dB


def _plain_balance(c, s):
    sc = s["logits"].float() * _scales(c)[0]
    T, E, k = c["T"], c["E"], c["k"]
    valid = torch.ones(T, dtype=torch.bool, device=sc.device) if s["mask"] is None else s["mask"]
    counts = torch.zeros(E + 1, dtype=torch.int32, device=sc.device)
    counts.scatter_add_(0, s["idx"].long().flatten(), valid[:, None].expand(T, k).int().flatten())
    n = valid.sum()
    counts[E] = n
    zero = torch.zeros((), device=sc.device)
    P = torch.where(valid[:, None], _probs(c, sc), zero).sum(0)
    z = torch.where(valid, _lse(sc) ** 2, zero).sum()
    nf = n.clamp(min=1).float()
    bal = (counts[:E].float() / (nf * k) * (P / nf)).sum() * E
    return {"counts": counts, "prob_sum": P, "losses": torch.stack([bal, z / nf])}


def _plain_router(c, s):
    dt = s["logits"].dtype
    E, k = c["E"], c["k"]
    ls, rs = _scales(c)
    sc = s["logits"].float() * ls
    idx = s["idx"].long()
    g = s["dw"] * rs
    if c["gating"] == "sigmoid":
        raw = 1.0 / (1.0 + torch.exp(-sc.gather(1, idx)))
        if c["norm"] and k > 1:
            S = raw.sum(-1, keepdim=True) + 1e-20
            g = (g - (g * raw).sum(-1, keepdim=True) / S) / S
        ds = torch.zeros_like(sc).scatter_add(1, idx, g * raw * (1.0 - raw))
    elif c["gating"] == "topk_softmax" or (c["norm"] and s["eb"] is None):
        l = sc.gather(1, idx)
        e = torch.exp(l - l.amax(-1, keepdim=True))
        w = e / e.sum(-1, keepdim=True)
        ds = torch.zeros_like(sc).scatter_add(1, idx, w * (g - (g * w).sum(-1, keepdim=True)))
    else:
        p = _probs(c, sc)
        if c["norm"]:
            v = p.gather(1, idx) + (0.0 if s["eb"] is None else s["eb"][idx])
            S = v.sum(-1, keepdim=True)
            g = (g - (g * v).sum(-1, keepdim=True) / S) / S
        dp = torch.zeros_like(sc).scatter_add(1, idx, g)
        ds = p * (dp - (dp * p).sum(-1, keepdim=True))
    # the balance and z losses
    n = s["counts"][E].clamp(min=1).float()
    f = s["counts"][:E].float() * (s["coefs"][0] * E / (k * n * n))
    q = _probs(c, sc)
    d = q * (f - (q * f).sum(-1, keepdim=True))
    if c["gating"] == "sigmoid":
        d = d / (1.0 + torch.exp(sc))  # dq through each sigmoid: q (1 - sigmoid)
    p = torch.exp(sc - _lse(sc)[:, None])
    ds = ds + d + (2.0 * s["coefs"][1] / n) * _lse(sc)[:, None] * p
    if s["mask"] is not None:
        ds = torch.where(s["mask"][:, None], ds, torch.zeros((), device=ds.device))
    return (ds * ls).to(dt)


# ----------------------------------------------------------------- exact --

def exact(case, seed):
    """The definitions in float64; gradients by differentiating them."""
    c = case
    s = prepare(c, seed)
    if c["op"] in ("balance", "router"):
        l = s["logits"].double().requires_grad_(True)
        ls, rs = _scales(c)
        sc = l * ls
        idx = s["idx"].long()
        rows = torch.arange(c["T"], device=l.device) if s["mask"] is None else s["mask"].nonzero()[:, 0]
        if c["op"] == "balance":
            counts = torch.bincount(idx[rows].flatten(), minlength=c["E"]).to(torch.int32)
            counts = torch.cat([counts, torch.tensor([len(rows)], dtype=torch.int32, device=l.device)])
            n = max(1, len(rows))
        else:
            counts, n = s["counts"], max(1, int(s["counts"][-1]))
        v = sc[rows]
        q = torch.sigmoid(v)
        q = q / q.sum(1, keepdim=True) if c["gating"] == "sigmoid" else torch.softmax(v, 1)
        P = q.sum(0)
        bal = c["E"] * torch.dot(counts[:-1].double() / (n * c["k"]), P / n)
        z = torch.logsumexp(v, 1).square().sum() / n
        if c["op"] == "balance":
            return {"counts": counts, "prob_sum": P.detach(), "losses": torch.stack([bal, z]).detach()}
        eb = torch.zeros(c["E"], device=l.device).double() if s["eb"] is None else s["eb"].double()
        pick = idx[rows]
        if c["gating"] == "sigmoid":
            w = torch.sigmoid(v).gather(1, pick)
            if c["norm"] and c["k"] > 1:
                w = w / (w.sum(1, keepdim=True) + 1e-20)
        elif c["gating"] == "topk_softmax":
            w = torch.softmax(v.gather(1, pick), 1)
        else:
            w = torch.softmax(v, 1).gather(1, pick) + eb[pick]
            if c["norm"]:
                w = w / w.sum(1, keepdim=True)
        loss = (rs * w * s["dw"].double()[rows]).sum() + s["coefs"][0] * bal + s["coefs"][1] * z
        return torch.autograd.grad(loss, l)[0]
    if c["op"] == "combine":
        w = s["w"].to(s["Y"].dtype).double().requires_grad_(True)
        dY = torch.empty(s["Y"].shape, dtype=torch.float64, device=s["Y"].device)
        dw = torch.empty(s["w"].shape, dtype=torch.float64, device=s["Y"].device)
        for r in range(c["k"]):
            at = s["inv"][:, r].long()
            y = s["Y"][at].double().requires_grad_(True)
            out = (w[:, r:r + 1] * y * s["dout"].double()).sum()
            gy, gw = torch.autograd.grad(out, [y, w])
            dY[at] = gy
            dw[:, r] = gw[:, r]
        return dY, dw
    x = s["x"].double().requires_grad_(True)
    A, B = s["A"].double().requires_grad_(True), s["B"].double().requires_grad_(True)
    y = torch.zeros(c["T"], c["N"], dtype=torch.float64, device=x.device)
    for a in range(c["G"]):
        rows = (s["ad"] == a).nonzero()[:, 0]
        if len(rows):
            y = y.index_add(0, rows, s["scale"][a].double() * ((x[rows] @ A[a].t()) @ B[a].t()))
    if c["op"] == "lora":
        return (s["y"].double() + y).detach()
    if not y.requires_grad:
        return s["dx"].double(), torch.zeros_like(A), torch.zeros_like(B)
    gx, gA, gB = torch.autograd.grad((y * s["dy"].double()).sum(), [x, A, B])
    return s["dx"].double() + gx, gA, gB
