"""The calls that take a gradient back through a layer of frozen quantised
experts: their inputs, their plain forms, their work and a float64 restatement
of their results.

Five operators, reached through ffai_amd.tuning:

  expert_matmul_backward  gradient of the rows of a grouped dequantising product
  activation_save         gated activation, its inputs kept in 8 bits (and read back)
  activation_backward     gradient of the activation from what was kept
  permute_backward        gradient of the rows sorted by expert, back in token order
  add_rmsnorm_backward    gradient of the residual add and RMS norm before the layer

Where `own` is false `run` computes them from elementary torch operations in
32 bits, otherwise through the library.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# Fields of a case by operator:
#   expert:  T tokens, E experts, k picks, N outputs and K inputs of the
#     projection (the gradient goes from N to K), bits, gs (group size), pair
#     (gate and up projections in one call), gather (the gradient's rows are the
#     tokens', picked through the plan, else one per sorted position), add
#     (added to another gradient), skew (spread of the experts' popularity)
#   save / act:  M rows, n columns, act ("swiglu", "gptoss", "geglu", "relu2"),
#     weights (act: rows with routing weights, back to token order), h (act:
#     the activation's value is asked for too)
#   permute:  T tokens, k picks, H hidden, add
#   norm:  T rows, H hidden, skip (a gradient of the residual beside the norm's)
EXPERT = dict(op="expert", gs=64, pair=False, gather=False, add=False, skew=0.5, dt="bf16")
ALPHA, LIMIT, EPS = 1.702, 7.0, 1e-6


def listed():
    return [
        # a short batch on few large experts, six rows each: the down projection,
        # whose gradient comes in token order; bound by the experts' bytes
        dict(EXPERT, name="expert_t48_h2880", T=48, E=32, k=4, N=2880, K=2880, bits=4, gather=True),
        # an odd-length sequence on many small 3-bit experts, f16, gate and up
        # together, added to the adapters' gradient
        dict(EXPERT, name="expert_t777_e256_3bit", T=777, E=256, k=8, N=512, K=2048, bits=3, pair=True, add=True, dt="f16"),
        # a training batch of 4096 tokens on 128 experts, gate and up together
        dict(EXPERT, name="expert_t4096_e128", T=4096, E=128, k=8, N=768, K=2048, bits=4, pair=True),
        # a small f32 layer, 6-bit codes in groups of 32
        dict(EXPERT, name="expert_t200_f32", T=200, E=8, k=2, N=512, K=1024, bits=6, gs=32, gather=True, dt="f32"),
        # the forward of a short batch on few large experts
        dict(name="save_m148_n2880", op="save", M=148, n=2880, act="gptoss", dt="bf16"),
        # the forward of a training batch: 4096 tokens, 8 experts each
        dict(name="save_m32768_n768", op="save", M=32768, n=768, act="swiglu", dt="bf16"),
        # an odd-length sequence, f16, the value asked for again
        dict(name="act_m1998_n512", op="act", M=1998, n=512, act="geglu", weights=True, h=True, dt="f16"),
        # the backward of the training batch
        dict(name="act_m32768_n768", op="act", M=32768, n=768, act="swiglu", weights=True, h=False, dt="bf16"),
        # a short odd batch
        dict(name="permute_t37_h2880", op="permute", T=37, k=4, H=2880, add=True, dt="bf16"),
        # the training batch, beside the router's and the shared expert's gradient
        dict(name="permute_t4096_h2048", op="permute", T=4096, k=8, H=2048, add=True, dt="bf16"),
        # a short f32 batch: few rows share the weight's gradient
        dict(name="norm_t50_h1024_f32", op="norm", T=50, H=1024, skip=False, dt="f32"),
        # two sequences of 4096 tokens: many rows meet in the weight's gradient
        dict(name="norm_t8192_h2048", op="norm", T=8192, H=2048, skip=True, dt="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    top = [work(c) for c in listed()]
    while True:
        op = rng.choice(["expert", "expert", "expert", "save", "act", "act", "permute", "norm"])
        dt = rng.choice(["bf16", "bf16", "f16", "f32"])
        act = rng.choice(["swiglu", "swiglu", "gptoss", "geglu", "relu2"])
        if op == "expert":
            E = rng.choice([1, 8, 32, 60, 64, 128, 256, rng.randint(2, 200)])
            gs = rng.choice([32, 64, 64, 128])
            pair = rng.random() < 0.5
            c = dict(EXPERT, T=_log(rng, 1, 4096), E=E, k=rng.randint(1, min(E, 8)), N=32 * _log(rng, 2, 92),
                     K=gs * _log(rng, 2, 3000 // gs), bits=rng.choice([2, 3, 4, 4, 5, 6, 8]), gs=gs, pair=pair,
                     gather=not pair and rng.random() < 0.5, add=rng.random() < 0.3,
                     skew=rng.choice([0.0, 0.5, 1.0]), dt=dt)
            if dt == "f32" and work(c)["flops"] > 0.1 * max(w["flops"] for w in top):
                continue
        elif op == "save":
            c = dict(op=op, M=_log(rng, 1, 65536), n=32 * _log(rng, 2, 128), act=act, dt=dt)
        elif op == "act":
            c = dict(op=op, M=_log(rng, 1, 65536), n=32 * _log(rng, 2, 128), act=act, weights=rng.random() < 0.7,
                     h=rng.random() < 0.3, dt=dt)
        elif op == "permute":
            c = dict(op=op, T=_log(rng, 1, 8192), k=rng.randint(1, 10), H=8 * _log(rng, 8, 512), add=rng.random() < 0.7, dt=dt)
        else:
            c = dict(op=op, T=_log(rng, 1, 16384), H=8 * _log(rng, 8, 1024), skip=rng.random() < 0.7, dt=dt)
        w = work(c)
        most = [v for v, l in zip(top, listed()) if l["op"] == op]
        if all(w[m] <= max(v[m] for v in most) for m in w):
            return c


def work(case):
    c = case
    es = 4 if c["dt"] == "f32" else 2
    if c["op"] == "expert":  # the used experts, the gradient's rows, the plan in; the rows' gradient out
        M, P = c["T"] * c["k"], 2 if c["pair"] else 1
        used = c["E"] * (1.0 - (1.0 - c["k"] / c["E"]) ** c["T"])
        stack = used * c["N"] * c["K"] * (c["bits"] / 8 + 2 * es / c["gs"])
        rows = (c["T"] if c["gather"] else M) * c["N"] * es
        return {"bytes": P * (stack + rows) + (2 if c["add"] else 1) * M * c["K"] * es + 4 * c["E"] + (4 * M if c["gather"] else 0),
                "flops": 2.0 * P * M * c["N"] * c["K"]}
    if c["op"] in ("save", "act"):
        parts = 1 if c["act"] == "relu2" else 2
        el, kept = c["M"] * c["n"], parts * c["M"] * c["n"] * (1 + 1 / 32)
        if c["op"] == "save":  # projections in; value, codes and scales out; codes and scales in, values out
            return {"bytes": el * es * (2 * parts + 1) + 2 * kept, "flops": 20 * el}
        # codes, scales and the value's gradient in; the projections' gradients (and value) out
        return {"bytes": el * es * (1 + parts + c["h"]) + kept + 12 * c["M"] * c["weights"], "flops": 30 * el}
    if c["op"] == "permute":
        return {"bytes": c["T"] * c["H"] * es * (c["k"] + 1 + c["add"]) + 4 * c["T"] * c["k"], "flops": c["T"] * c["H"] * c["k"]}
    return {"bytes": c["T"] * c["H"] * es * (3 + c["skip"]) + c["H"] * (es + 4), "flops": 12 * c["T"] * c["H"]}


# ---------------------------------------------------------------- inputs --

def _randn(gen, *shape, std=1.0):
    return torch.randn(*shape, device="cuda", generator=gen).mul_(std)


def _plan(c, gen):
    """perm and offsets of T tokens with k picks each, experts of unequal popularity."""
    T, E, k = c["T"], c["E"], c["k"]
    score = _randn(gen, E, std=c["skew"]) - torch.log(-torch.log(torch.rand(T, E, device="cuda", generator=gen).clamp_(1e-9, 1 - 1e-7)))
    idx = score.topk(k).indices.flatten()
    perm = idx.argsort(stable=True)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = torch.bincount(idx, minlength=E).cumsum(0)
    return perm.to(torch.int32), offsets.to(torch.int32)


def _stack(c, gen):
    """A quantised stack: codes, scales and biases of weights around zero."""
    E, N, K, bits, dt = c["E"], c["N"], c["K"], c["bits"], DTYPES[c["dt"]]
    w = torch.randint(-2 ** 31, 2 ** 31, (E, N, K * bits // 32), device="cuda", generator=gen, dtype=torch.int64).to(torch.int32)
    s = torch.empty(E, N, K // c["gs"], device="cuda").uniform_(0.5, 1.5, generator=gen).mul_(3.0 * N ** -0.5 / 2 ** bits)
    b = s * (-(2 ** bits - 1) / 2) + _randn(gen, *s.shape, std=0.05 * N ** -0.5)
    return w, s.to(dt), b.to(dt)


def _keep(v):
    """8-bit codes and exponent bytes of blocks of 32 along the last axis: the
    least exponent e that keeps a block's largest below 127.5 steps of 2^(e - 133)."""
    blocks = v.float().reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    top = blocks.abs().amax(-1).view(torch.int32)
    e = (top + 0x10000) >> 23
    codes = torch.round(torch.ldexp(blocks, (133 - e)[..., None]))
    return codes.reshape(v.shape), e


def _kept(codes, e):
    """The values they stand for."""
    blocks = codes.float().reshape(*codes.shape[:-1], codes.shape[-1] // 32, 32)
    return torch.ldexp(blocks, (e.to(torch.int32) - 133)[..., None]).reshape(codes.shape)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dt"]]
    s = dict(case=c)
    if c["op"] == "expert":
        T, k, N, K = c["T"], c["k"], c["N"], c["K"]
        M = T * k
        s["perm"], s["offsets"] = _plan(c, gen)
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        s["stacks"] = [_stack(c, gen) for _ in range(2 if c["pair"] else 1)]
        s["dy"] = [_randn(gen, T if c["gather"] else M, N, std=0.01).to(dt) for _ in s["stacks"]]
        s["dx"] = _randn(gen, M, K, std=0.01).to(dt) if c["add"] else None
        if own:
            from ffai_amd.layer import StackedExperts
            s["projs"] = [StackedExperts(*t, c["bits"], c["gs"]) for t in s["stacks"]]
    elif c["op"] in ("save", "act"):
        parts = 1 if c["act"] == "relu2" else 2
        # a few columns far larger than the others, as activations have them
        wide = torch.exp(_randn(gen, parts, 1, c["n"], std=0.7))
        v = (_randn(gen, parts, c["M"], c["n"], std=1.2) * wide).to(dt)
        if c["op"] == "save":
            s["v"] = v
        else:
            codes, e = _keep(v)
            s["codes"], s["e"] = codes.to(torch.int8), e.to(torch.uint8)
            s["dh"] = _randn(gen, c["M"], c["n"], std=0.01).to(dt)
            s["w"] = s["perm"] = None
            if c["weights"]:
                s["w"] = torch.rand(c["M"], device="cuda", generator=gen)
                s["perm"] = torch.rand(c["M"], device="cuda", generator=gen).argsort().to(torch.int32)
        if own:
            from ffai_amd import _lib, tuning
            s["act"] = {"swiglu": _lib.MOE_ACT_SWIGLU, "gptoss": _lib.MOE_ACT_GPTOSS, "geglu": _lib.MOE_ACT_GEGLU,
                        "relu2": _lib.MOE_ACT_RELU2}[c["act"]]
            if c["op"] == "act":
                s["kept"] = tuning.Checkpoint8(s["codes"], s["e"])
    elif c["op"] == "permute":
        T, k, H = c["T"], c["k"], c["H"]
        s["inv"] = torch.rand(T * k, device="cuda", generator=gen).argsort().to(torch.int32).reshape(T, k)
        s["dX"] = _randn(gen, T * k, H, std=0.01).to(dt)
        s["dx"] = _randn(gen, T, H, std=0.01).to(dt) if c["add"] else None
    else:
        T, H = c["T"], c["H"]
        s["r"] = (_randn(gen, T, H) * torch.exp(_randn(gen, T, 1, std=0.5))).to(dt)
        s["w"] = (1.0 + _randn(gen, H, std=0.2)).to(dt)
        s["dn"] = _randn(gen, T, H, std=0.01).to(dt)
        s["dr"] = _randn(gen, T, H, std=0.01).to(dt) if c["skip"] else None
    return s


# ------------------------------------------------------------------- run --

def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from ffai_amd import tuning
    c = s["case"]
    if c["op"] == "expert":
        p, dy = s["projs"], s["dy"]
        return tuning.expert_matmul_backward(p[0], dy[0], s["offsets"], perm=s["perm"] if c["gather"] else None, top_k=c["k"],
                                             proj2=p[1] if c["pair"] else None, dy2=dy[1] if c["pair"] else None, dx=s["dx"],
                                             out=None if s["dx"] is None else torch.empty_like(s["dx"]))
    if c["op"] == "save":
        gate, up = (None, s["v"][0]) if c["act"] == "relu2" else (s["v"][0], s["v"][1])
        h, kept = tuning.activation_save(gate, up, s["act"], ALPHA, LIMIT)
        return h, kept.restore(up.dtype)
    if c["op"] == "act":
        g = tuning.activation_backward(s["kept"], s["dh"], s["act"], ALPHA, LIMIT, topk_weight=s["w"], perm=s["perm"], want_h=c["h"])
        return {"d_gate": g.d_gate, "d_up": g.d_up, "d_weight": g.d_weight if c["weights"] else None, "h": g.h}
    if c["op"] == "permute":
        return tuning.permute_backward(s["dX"], s["inv"], dx=s["dx"], out=None if s["dx"] is None else torch.empty_like(s["dx"]))
    return tuning.add_rmsnorm_backward(s["r"], s["w"], s["dn"], EPS, d_residual=s["dr"])


def _dequantised(w, sc, b, bits, gs):
    """float32 weights of a stack of packed codes."""
    E, N, words = w.shape
    K = words * 32 // bits
    at = torch.arange(K, device=w.device) * bits
    lo, sh = at >> 5, (at & 31).to(torch.int32)
    rest = torch.where(sh == 0, -1, (1 << (32 - sh.long())) - 1).to(torch.int32)  # the bits a word has left
    q = (w[..., lo] >> sh) & rest
    if 32 % bits:  # a code may end in the next word
        hi = (lo + 1).clamp(max=words - 1)
        q = q | torch.where(sh + bits > 32, (w[..., hi] << 1) << (31 - sh), torch.zeros((), dtype=torch.int32, device=w.device))
    q = (q & (2 ** bits - 1)).float().reshape(E, N, K // gs, gs)
    return (q * sc.float()[..., None] + b.float()[..., None]).reshape(E, N, K)


def _act(c, g, u):
    """(value, d value / d gate, d value / d up) of the activation; gelu's value
    is rounded to the rows' type before the product."""
    if c["act"] == "relu2":
        r = u.clamp(min=0.0)
        return r * r, None, 2.0 * r
    if c["act"] == "gptoss":
        gc, uc = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        sg = 1.0 / (1.0 + torch.exp(-ALPHA * gc))
        a = gc * sg
        da = sg + ALPHA * a * (1.0 - sg)
        return a * (uc + 1.0), da * (uc + 1.0) * (g <= LIMIT), a * (u.abs() <= LIMIT)
    if c["act"] == "geglu":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))
        a = 0.5 * g * (1.0 + t)
        da = 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * g * g)
        a = a.to(DTYPES[c["dt"]]).float()
        return a * u, da * u, a
    sg = 1.0 / (1.0 + torch.exp(-g))
    a = g * sg
    return a * u, (sg + a * (1.0 - sg)) * u, a


def _plain(s):
    c = s["case"]
    dt = DTYPES[c["dt"]]
    if c["op"] == "expert":
        # every expert's rows in a table of the longest one's length
        M, E = c["T"] * c["k"], c["E"]
        offsets = s["offsets"].long()
        p = torch.arange(M, device=offsets.device)
        e = torch.searchsorted(offsets[1:], p, right=True)
        slot = p - offsets[e]
        row = s["perm"].long() // c["k"] if c["gather"] else p
        out = 0.0 if s["dx"] is None else s["dx"].float()

        def product(stack, dy):
            table = torch.zeros(E, s["most"], c["N"], device=dy.device)
            table[e, slot] = dy[row].float()
            return torch.bmm(table, _dequantised(*stack, c["bits"], c["gs"]))[e, slot]

        out = out + product(s["stacks"][0], s["dy"][0])
        if c["pair"]:
            out = out + product(s["stacks"][1], s["dy"][1])
        return out.to(dt)
    if c["op"] == "save":
        v = s["v"].float()
        h = _act(c, None if c["act"] == "relu2" else v[0], v[-1])[0].to(dt)
        return h, _kept(*_keep(v)).to(dt)
    if c["op"] == "act":
        v, dh = _kept(s["codes"], s["e"]), s["dh"].float()
        h, hg, hu = _act(c, None if c["act"] == "relu2" else v[0], v[-1])
        dw = None
        r = dh
        if c["weights"]:
            perm = s["perm"].long()
            dw = torch.empty_like(s["w"])
            dw[perm] = (dh * h).sum(-1)
            r = s["w"].to(dt).float()[perm][:, None] * dh
        return {"d_gate": None if hg is None else (r * hg).to(dt), "d_up": (r * hu).to(dt), "d_weight": dw,
                "h": h.to(dt) if c["h"] else None}
    if c["op"] == "permute":
        out = s["dX"].float()[s["inv"].long()].sum(1)
        return (out if s["dx"] is None else out + s["dx"].float()).to(dt)
    r, w, dn = s["r"].float(), s["w"].float(), s["dn"].float()
    inv = 1.0 / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS)
    n = r * inv
    g = dn * w
    d = inv * (g - n * (g * n).mean(-1, keepdim=True))
    return (d if s["dr"] is None else d + s["dr"].float()).to(dt), (dn * n).sum(0)


# ----------------------------------------------------------------- exact --

def _function(c, g, u):
    """The activation in float64, as a function that autograd differentiates."""
    if c["act"] == "relu2":
        return torch.where(u > 0, u, torch.zeros_like(u)) ** 2
    if c["act"] == "gptoss":
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        return g * torch.sigmoid(ALPHA * g) * (u + 1)
    if c["act"] == "geglu":
        a = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        a = a + (a.detach().to(DTYPES[c["dt"]]).double() - a.detach())  # the value is rounded, the slope is gelu's
        return a * u
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    """The definitions in float64; gradients by differentiating them."""
    c = case
    s = prepare(c, seed)
    if c["op"] == "expert":
        at = s["offsets"].tolist()
        bits, gs = c["bits"], c["gs"]
        value = 2.0 ** torch.arange(bits, device="cuda", dtype=torch.float64)
        out = torch.zeros(c["T"] * c["k"], c["K"], dtype=torch.float64, device="cuda")
        if s["dx"] is not None:
            out += s["dx"].double()
        for (w, sc, b), dy in zip(s["stacks"], s["dy"]):
            for e in range(c["E"]):
                if at[e + 1] == at[e]:
                    continue
                here = torch.arange(at[e], at[e + 1], device="cuda")
                rows = torch.div(s["perm"][here].long(), c["k"], rounding_mode="floor") if c["gather"] else here
                stream = (w[e][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
                codes = stream.reshape(c["N"], c["K"], bits).double() @ value
                W = codes * sc[e].double().repeat_interleave(gs, 1) + b[e].double().repeat_interleave(gs, 1)
                out[here] += dy[rows].double() @ W
        return out
    if c["op"] == "save":
        v = s["v"].double()
        h = _function(c, v[0], v[-1])
        blocks = v.reshape(-1, 32)
        step = torch.full((len(blocks), 1), 2.0 ** -133, dtype=torch.float64, device="cuda")
        top = blocks.abs().amax(1, keepdim=True)
        # the least power of two of which 127.5 exceed the largest
        step = torch.maximum(step, torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-60) / 127.5)) + 1))
        step = torch.where(top < 127.5 * step / 2, step / 2, torch.where(top >= 127.5 * step, step * 2, step))
        return h, (torch.round(blocks / step) * step).reshape(v.shape)
    if c["op"] == "act":
        steps = torch.exp2(s["e"].double() - 133).repeat_interleave(32, -1)
        v = (s["codes"].double() * steps).requires_grad_(True)
        h = _function(c, v[0], v[-1])
        dh = s["dh"].double()
        r, dw = dh, None
        if c["weights"]:
            perm = s["perm"].long()
            r = s["w"].to(DTYPES[c["dt"]]).double()[perm][:, None] * dh
            dw = torch.zeros(c["M"], dtype=torch.float64, device="cuda").index_add(0, perm, (h.detach() * dh).sum(1))
        d = torch.autograd.grad((h * r).sum(), v)[0]
        return {"d_gate": None if c["act"] == "relu2" else d[0], "d_up": d[-1], "d_weight": dw, "h": h.detach() if c["h"] else None}
    if c["op"] == "permute":
        out = torch.zeros(c["T"], c["H"], dtype=torch.float64, device="cuda") if s["dx"] is None else s["dx"].double()
        for r in range(c["k"]):
            out = out + s["dX"][s["inv"][:, r].long()].double()
        return out
    r, w = s["r"].double().requires_grad_(True), s["w"].double().requires_grad_(True)
    y = r / torch.sqrt((r * r).sum(1, keepdim=True) / c["H"] + EPS) * w
    loss = (y * s["dn"].double()).sum()
    if s["dr"] is not None:
        loss = loss + (r * s["dr"].double()).sum()
    return torch.autograd.grad(loss, [r, w])
