"""Tuning and adapter entry points on the GPU against float64 restatements.

Tolerances follow from the arithmetic: a result rounded to type t is off by at
most eps(t)/2 of its value, a sum of n fp32 products by at most (n + c) 2^-24
of the sum of their magnitudes (c: the few roundings of its factors), and a
factor kept as two 16-bit parts by 2^-17 of itself."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd._lib import check  # noqa: E402
from ffai_amd.layer import MoEGatingMode, MoERouter, moe_dtype  # noqa: E402

U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SOFT, PICK, SIGM = MoEGatingMode.softmaxThenTopK, MoEGatingMode.topKThenSoftmax, MoEGatingMode.sigmoidTopK


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    _lib.load()
    yield
    torch.cuda.synchronize()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cuda(t):
    return None if t is None else t.cuda()


def close(got, ref, tol, what):
    """|got - ref| <= half a step of got's type + tol, elementwise, in float64;
    NaN and infinities have to match."""
    half = torch.finfo(got.dtype).eps / 2
    # below the smallest normal value the steps stay eps * that value apart, so
    # a rounding is off by up to half of it (f16: 2^-14 2^-10 / 2 = 2^-25)
    low = torch.finfo(got.dtype).smallest_normal * half
    got, ref = got.double().cpu(), ref.double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64)
    bound = half * (ref.abs() + tol) + tol + low + torch.finfo(torch.float32).tiny
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN pattern"
    bad = ((got - ref).abs() > bound) & fin
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{((got - ref).abs() / bound)[fin].max():.3g} of the bound")
    inf = ~fin & ~torch.isnan(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities"


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# --------------------------------------------------------------- routers --

def rows(T, E, k, dt, seed, mask="none", std=1.0):
    g = gen(seed)
    logits = (torch.randn(T, E, generator=g) * std + torch.randn(E, generator=g)).to(dt)
    idx = torch.rand(T, E, generator=g).topk(k).indices.to(torch.int32)
    m = {"none": None, "some": torch.rand(T, generator=g) < 0.6, "all": torch.zeros(T, dtype=torch.bool),
         "u8": (torch.rand(T, generator=g) < 0.5).to(torch.uint8) * 7}[mask]
    return logits, idx, m


def probs64(s, gating):
    if gating == SIGM:
        q = torch.sigmoid(s)
        return q / q.sum(1, keepdim=True)
    return torch.softmax(s, 1)


def losses64(s, counts, n, k, gating):
    E = s.shape[1]
    n = max(1, n)
    bal = E * (counts.double() / (k * n) * probs64(s, gating).sum(0) / n).sum()
    return bal, torch.logsumexp(s, 1).square().sum() / n


def counts_of(idx, m, E):
    on = torch.ones(len(idx), dtype=torch.bool) if m is None else m.bool()
    pick = idx[on].flatten().long()
    pick = pick[(pick >= 0) & (pick < E)]
    return torch.cat([torch.bincount(pick, minlength=E), on.sum()[None]]).to(torch.int32), on


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,E,k,gating,mask", [
    (1, 8, 2, SOFT, "none"), (1, 5, 5, SIGM, "all"), (3, 1, 1, SOFT, "none"), (64, 32, 4, PICK, "none"),
    (37, 60, 8, SIGM, "some"), (333, 128, 6, SIGM, "u8"), (1000, 256, 8, SOFT, "some"), (700, 512, 64, SOFT, "none"),
    (4097, 8, 2, SOFT, "some"), (515, 509, 3, PICK, "some"), (9001, 128, 8, SOFT, "all"), (129, 9, 9, SOFT, "none"),
])
def test_balance_loss(dt, T, E, k, gating, mask):
    lg, idx, m = rows(T, E, k, dt, T * 31 + E, mask)
    r = MoERouter(E, k, gating, True, None, 0.5 if E == 60 else 1.0)
    b = tuning.balance_loss(r, lg.cuda(), idx.cuda(), mask=cuda(m))
    counts, on = counts_of(idx, m, E)
    s = lg.double() * r.logitScale
    n = int(on.sum())
    P = probs64(s[on], gating).sum(0)
    assert torch.equal(b.counts.cpu(), counts)
    # p is off by a few roundings (exp, the row's sum of E terms, the divide)
    c = (E + 16) * U
    close(b.prob_sum, P, P * (c + (n + 8) * U), "P")
    bal, z = losses64(s[on], counts[:-1], n, k, gating) if n else (torch.zeros(()), torch.zeros(()))
    lse = torch.logsumexp(s[on], 1).abs()
    zt = (2 * lse * (c + lse * 4 * U)).sum() / max(1, n) + z * (n + 8) * U
    tol = torch.stack([torch.as_tensor(bal * (c + (n + 8) * U)).double(), torch.as_tensor(zt).double()])
    close(b.losses, torch.stack([torch.as_tensor(bal).double(), torch.as_tensor(z).double()]), tol, "losses")


def test_balance_loss_edge_rows():
    """Masked rows may hold anything; a row of -inf only has no probability; ids
    out of range are not counted and one that appears twice counts twice."""
    E, k = 16, 4
    for T in (40, 3000):
        lg, idx, _ = rows(T, E, k, F32, 3)
        m = torch.ones(T, dtype=torch.bool)
        m[::3] = False
        lg[0] = float("nan")
        lg[3] = float("inf")
        lg[1] = float("-inf")
        lg[4, 5:] = float("-inf")
        idx[2] = torch.tensor([16, -1, 7, 7])
        r = MoERouter(E, k)
        b = tuning.balance_loss(r, lg.cuda(), idx.cuda(), mask=m.cuda())
        counts, on = counts_of(idx, m, E)
        assert torch.equal(b.counts.cpu(), counts)
        on2 = on.clone()
        on2[1] = False
        s, n = lg.double()[on2], int(on.sum())
        P = torch.softmax(s, 1).sum(0)
        close(b.prob_sum, P, P * (n + 40) * U, "P")
        bal = E * (counts[:-1].double() / (k * n) * P / n).sum()
        lse = torch.logsumexp(s, 1)
        z = lse.square().sum() / n
        close(b.losses, torch.stack([bal, z]), torch.stack([bal, z + lse.abs().mean()]) * (n + 60) * U, "losses")
        lg[2, 3] = float("nan")
        b = tuning.balance_loss(r, lg.cuda(), idx.cuda(), mask=m.cuda())
        assert torch.isnan(b.losses).all() and torch.isnan(b.prob_sum).all()


def weights64(s, idx, gating, norm, eb, rs, es):
    """MoERouter's weights of given picks (ids out of range: no weight)."""
    ok = (idx >= 0) & (idx < s.shape[1])
    at = idx.clamp(0, s.shape[1] - 1).long()
    k = idx.shape[1]
    if gating == SIGM:
        w = torch.where(ok, torch.sigmoid(s).gather(1, at), 0.0)
        if norm and k > 1:
            w = w / (w.sum(1, keepdim=True) + 1e-20)
    elif gating == PICK or (norm and eb is None):
        w = torch.softmax(torch.where(ok, s.gather(1, at), float("-inf")), 1)
    else:
        w = torch.softmax(s, 1).gather(1, at)
        if eb is not None:
            w = w + eb.double()[at]
        w = torch.where(ok, w, 0.0)
        if norm:
            w = w / w.sum(1, keepdim=True)
    return w * rs * (1.0 if es is None else es.double()[at])


def router_ref(r, lg, idx, dw, counts, bal, z, m, eb, es):
    l = lg.double().requires_grad_(True)
    on = torch.ones(len(lg), dtype=torch.bool) if m is None else m.bool()
    s = l[on] * (r.logitScale or 1.0)
    loss = (s * 0.0).sum()
    if dw is not None:
        w = weights64(s, idx[on], r.gatingMode, r.normTopKProb, eb, r.routedScale or 1.0, es)
        loss = loss + (w * dw.double()[on]).sum()
    if counts is not None:
        b, zz = losses64(s, counts[:-1], int(counts[-1]), r.topK, r.gatingMode)
        loss = loss + bal * b + z * zz
    return torch.autograd.grad(loss, l)[0]


def router_tol(r, lg, idx, dw, counts, bal, z, eb, es):
    """A bound on the fp32 error of a row's gradients: every term is a product
    of factors that are off by (E + k + 24) roundings at most, and the terms'
    magnitudes are bounded by what multiplies them."""
    E, k = r.nExperts, r.topK
    s = lg.double() * (r.logitScale or 1.0)
    mag = torch.zeros(len(lg), 1, dtype=torch.float64)
    if dw is not None:
        g = dw.double().abs() * abs(r.routedScale or 1.0)
        if es is not None:
            g = g * es.double().abs().max()
        scale = 1.0
        if r.gatingMode == SIGM and r.normTopKProb and k > 1:
            scale = 1.0 / torch.sigmoid(s).gather(1, idx.clamp(0, E - 1).long()).sum(1, keepdim=True)
        elif r.gatingMode == SOFT and r.normTopKProb and eb is not None:
            v = torch.softmax(s, 1).gather(1, idx.clamp(0, E - 1).long()) + eb.double()[idx.clamp(0, E - 1).long()]
            scale = v.abs().sum(1, keepdim=True) / v.sum(1, keepdim=True).abs() ** 2
            scale = scale + 1.0 / v.sum(1, keepdim=True).abs()
        mag = mag + 2 * g.sum(1, keepdim=True) * scale
    if counts is not None:
        n = max(1, int(counts[-1]))
        mag = mag + 2 * abs(bal) * E / (k * n * n) * counts[:-1].max().double()
        mag = mag + 2 * abs(z) / n * (torch.logsumexp(s, 1, keepdim=True).abs() + 1)
    return mag.expand_as(s) * abs(r.logitScale or 1.0) * (E + k + 24) * U


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,E,k,gating,norm,bias,mask", [
    (1, 8, 2, SOFT, True, False, "none"), (5, 1, 1, SOFT, True, False, "none"), (2, 8, 8, SOFT, False, False, "none"),
    (33, 32, 4, PICK, True, False, "some"), (333, 128, 6, SIGM, True, True, "some"), (64, 128, 8, SOFT, True, True, "u8"),
    (100, 60, 8, SOFT, False, True, "none"), (77, 256, 8, SOFT, True, False, "some"), (19, 512, 64, SIGM, False, False, "none"),
    (130, 509, 10, PICK, False, False, "none"), (41, 9, 9, SIGM, True, False, "none"), (65, 64, 1, SIGM, True, False, "none"),
    (50, 128, 8, SOFT, True, False, "all"), (9000, 16, 2, SOFT, False, False, "some"),
])
def test_router_backward(dt, T, E, k, gating, norm, bias, mask):
    lg, idx, m = rows(T, E, k, dt, T + 7 * E + k, mask)
    g = gen(5)
    eb = torch.rand(E, generator=g) * 0.1 if bias else None
    es = torch.rand(E, generator=g) + 0.5 if E in (60, 128) else None
    r = MoERouter(E, k, gating, norm, cuda(eb), 0.7 if E == 256 else 1.0, 2.5 if gating == SIGM else 1.0, cuda(es))
    dw = torch.randn(T, k, generator=g)
    counts, on = counts_of(idx, m, E)
    for d, c, bal, z in [(dw, counts, 0.3, 0.2), (dw, None, 0.0, 0.0), (None, counts, 1.0, 0.0), (None, counts, 0.0, 1.0)]:
        got = tuning.router_backward(r, lg.cuda(), idx.cuda(), d_weight=cuda(d), counts=cuda(c), balance_coef=bal,
                                     z_coef=z, mask=cuda(m))
        ref = router_ref(r, lg, idx, d, c, bal, z, m, eb, es)
        close(got, ref, router_tol(r, lg, idx, d, c, bal, z, eb, es), f"d logits {bal} {z}")
        if m is not None:
            assert (got[~on.cuda()] == 0).all()


def test_router_backward_matches_differences():
    """The gradient against central differences of the float64 losses."""
    T, E, k = 6, 12, 3
    for gating, norm, bias in [(SOFT, True, False), (SOFT, False, False), (SOFT, True, True), (PICK, True, False),
                               (SIGM, True, False), (SIGM, False, False)]:
        lg, idx, _ = rows(T, E, k, F32, 11)
        g = gen(2)
        dw, eb = torch.randn(T, k, generator=g), (torch.rand(E, generator=g) if bias else None)
        r = MoERouter(E, k, gating, norm, cuda(eb), 0.9, 1.5)
        counts, _ = counts_of(idx, None, E)
        got = tuning.router_backward(r, lg.cuda(), idx.cuda(), dw.cuda(), counts.cuda(), 0.5, 0.25).double().cpu()

        def loss(l):
            s = l * 0.9
            b, z = losses64(s, counts[:-1], T, k, gating)
            return (weights64(s, idx, gating, norm, eb, 1.5, None) * dw.double()).sum() + 0.5 * b + 0.25 * z

        h = 1e-5
        for t, e in [(0, 0), (2, 7), (5, 11), (3, int(idx[3, 0])), (1, int(idx[1, 2]))]:
            d = torch.zeros(T, E, dtype=torch.float64)
            d[t, e] = h
            num = (loss(lg.double() + d) - loss(lg.double() - d)) / (2 * h)
            # truncation h^2 f''' / 6 with derivatives of order one, and the losses' rounding / h
            assert abs(float(num) - float(got[t, e])) <= 1e-8 + 1e-9 + 100 * U * (1 + abs(float(num)))


def test_router_backward_edge_rows():
    """-inf logits, rows of -inf only, masked NaN rows, ids twice and out of range."""
    T, E, k = 12, 24, 4
    for gating in (SOFT, PICK, SIGM):
        for norm in (True, False):
            lg, idx, _ = rows(T, E, k, F32, 8)
            m = torch.ones(T, dtype=torch.bool)
            m[5] = m[6] = False
            lg[5] = float("nan")
            lg[6] = float("inf")
            lg[2, 8:] = float("-inf")
            idx[2] = torch.tensor([1, 0, 3, 9])
            idx[3] = torch.tensor([4, 4, 2, 4])
            idx[4] = torch.tensor([24, 7, -1, 11])
            r = MoERouter(E, k, gating, norm)
            dw = torch.randn(T, k, generator=gen(1))
            counts, _ = counts_of(idx, m, E)
            got = tuning.router_backward(r, lg.cuda(), idx.cuda(), dw.cuda(), counts.cuda(), 0.5, 0.25, mask=m.cuda())
            ref = router_ref(r, lg, idx, dw, counts, 0.5, 0.25, m, None, None)
            keep = torch.ones(T, dtype=torch.bool)
            keep[5] = keep[6] = False
            assert (got.cpu()[~keep] == 0).all()
            # a -inf logit has a zero gradient (float64 gives NaN where 0 * inf meets)
            ref = torch.where(torch.isinf(lg), 0.0, ref)
            sl = torch.where(torch.isinf(lg), -30.0, lg.double())[keep]
            tol = router_tol(r, sl, idx[keep], dw[keep], counts, 0.5, 0.25, None, None)
            row = torch.arange(T)[keep]
            ok = torch.isfinite(ref[keep]).all(1)
            close(got.cpu()[keep][ok], ref[keep][ok], 4 * tol[ok], f"rows {row[ok].tolist()}")
            assert ok.sum() >= T - 3
    lg[1] = float("-inf")
    got = tuning.router_backward(r, lg.cuda(), idx.cuda(), dw.cuda(), counts.cuda(), 0.5, 0.25, mask=m.cuda())
    assert (got[1] == 0).all()
    lg[0, 3] = float("nan")
    got = tuning.router_backward(r, lg.cuda(), idx.cuda(), dw.cuda(), counts.cuda(), 0.5, 0.25, mask=m.cuda())
    assert torch.isnan(got[0]).any() and torch.isfinite(got[2:]).all()


def test_router_rows_at_odd_addresses():
    """A row image that starts off a 16-byte boundary takes the narrow loads."""
    T, E, k = 21, 32, 4
    lg, idx, _ = rows(T, E, k, BF16, 4)
    r = MoERouter(E, k)
    buf = torch.empty(T * E + 3, dtype=BF16, device="cuda")
    odd = buf[3:].view(T, E)
    odd.copy_(lg)
    counts, _ = counts_of(idx, None, E)
    b0, b1 = tuning.balance_loss(r, lg.cuda(), idx.cuda()), tuning.balance_loss(r, odd, idx.cuda())
    assert torch.equal(b0.counts, b1.counts) and same_bits(b0.losses, b1.losses)
    dw = torch.randn(T, k, generator=gen(9)).cuda()
    out = torch.full((T * E + 8,), 5.0, dtype=BF16, device="cuda")
    got = tuning.router_backward(r, odd, idx.cuda(), dw, counts.cuda(), 0.1, 0.1, out=out[1:1 + T * E].view(T, E))
    want = tuning.router_backward(r, lg.cuda(), idx.cuda(), dw, counts.cuda(), 0.1, 0.1)
    assert same_bits(got, want) and out[0] == 5 and (out[1 + T * E:] == 5).all()


# --------------------------------------------------------------- combine --

@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,H,k", [(1, 8, 1), (1, 2048, 8), (37, 2880, 4), (5, 2056, 9), (130, 64, 10), (3, 8192, 2), (2, 72, 64)])
def test_unpermute_backward(dt, T, H, k):
    g = gen(T + H + k)
    M = T * k
    inv = torch.randperm(M, generator=g).to(torch.int32)
    w = torch.rand(T, k, generator=g)
    Y, d = torch.randn(M, H, generator=g).to(dt), torch.randn(T, H, generator=g).to(dt)
    dY, dw = tuning.unpermute_backward(d.cuda(), Y.cuda(), inv.cuda(), w.cuda())
    wr = w.to(dt).double()
    want = torch.empty(M, H, dtype=torch.float64)
    want[inv.long()] = (wr[:, :, None] * d.double()[:, None]).reshape(M, H)
    close(dY, want, 0.0, "dY")
    rowsY = Y.double()[inv.long()].view(T, k, H)
    close(dw, (rowsY * d.double()[:, None]).sum(-1), (rowsY * d.double()[:, None]).abs().sum(-1) * (H + 2) * U, "dw")
    # in place: the same bits
    y2 = Y.cuda()
    a, b = tuning.unpermute_backward(d.cuda(), y2, inv.cuda().view(T, k), w.cuda(), dY=y2)
    assert a.data_ptr() == y2.data_ptr() and same_bits(a, dY) and same_bits(b, dw)


def test_unpermute_backward_dropped_positions():
    """Positions past the plan have no row and a zero weight gradient, and rows
    that no position names stay as they were; dY is optional in the C ABI."""
    T, H, k = 9, 64, 3
    g = gen(1)
    inv = torch.arange(T * k, dtype=torch.int32).flip(0).contiguous()
    inv[4], inv[20] = 10 ** 6, -1
    Y, d, w = torch.randn(T * k, H, generator=g), torch.randn(T, H, generator=g), torch.rand(T, k, generator=g)
    dY = torch.full((T * k, H), 7.0).cuda()
    dY, dw = tuning.unpermute_backward(d.cuda(), Y.cuda(), inv.cuda(), w.cuda(), dY=dY)
    assert dw.flatten()[4] == 0 and dw.flatten()[20] == 0 and (dw != 0).sum() == T * k - 2
    assert (dY[T * k - 1 - 4] == 7).all() and (dY[T * k - 1 - 20] == 7).all() and (dY == 7).all(1).sum() == 2
    only = torch.empty(T, k, device="cuda")
    dc, Yc, ic, wc = d.cuda(), Y.cuda(), inv.cuda(), w.cuda()
    check(_lib.load().moe_unpermute_backward(dc.data_ptr(), Yc.data_ptr(), ic.data_ptr(), wc.data_ptr(), T, H, k, None,
                                             only.data_ptr(), moe_dtype(F32),
                                             C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert same_bits(only, dw)


# -------------------------------------------------------------- adapters --

def lora_case(T, K, N, R, G, dt, seed, kind="requests", bstd=0.05):
    g = gen(seed)
    x = torch.randn(T, K, generator=g).to(dt)
    A = (torch.randn(G, R, K, generator=g) * K ** -0.5).to(dt)
    B = (torch.randn(G, N, R, generator=g) * bstd).to(dt)
    scale = torch.rand(G, generator=g) * 1.5 + 0.5
    if kind == "each":
        ad = torch.randint(-1, G, (T,), generator=g)
    elif kind == "none":
        ad = torch.full((T,), -1)
    elif kind == "one":
        ad = torch.full((T,), G - 1)
    else:
        n = max(1, min(T, 5))
        ad = torch.randint(-1, G, (n,), generator=g)[torch.arange(T) * n // T]
    return x, A, B, scale, ad.to(torch.int32)


def split_err(dt):
    return 0.0 if dt == F32 else 2.0 ** -17


def lora_ref(x, A, B, scale, ad):
    """The adapters' rows in float64 and a bound on their fp32 error."""
    T, N = x.shape[0], B.shape[1]
    y, mag = torch.zeros(T, N, dtype=torch.float64), torch.zeros(T, N, dtype=torch.float64)
    for a in range(A.shape[0]):
        r = (ad == a).nonzero()[:, 0]
        if len(r):
            s = 1.0 if scale is None else float(scale[a])
            y[r] = s * ((x[r].double() @ A[a].double().t()) @ B[a].double().t())
            mag[r] = s * ((x[r].double().abs() @ A[a].double().abs().t()) @ B[a].double().abs().t())
    return y, mag * ((x.shape[1] + A.shape[1] + 16) * U + split_err(x.dtype))


SHAPES = [
    (1, 8, 8, 8, 1, "one"), (1, 2048, 768, 16, 64, "each"), (2, 64, 136, 24, 3, "each"), (16, 256, 64, 32, 2, "requests"),
    (17, 200, 264, 16, 40, "each"), (64, 512, 512, 16, 64, "each"), (100, 1032, 72, 40, 7, "each"), (15, 128, 2880, 64, 4, "requests"),
    (130, 2880, 128, 128, 5, "requests"), (333, 96, 328, 8, 1, "one"), (700, 320, 256, 72, 9, "requests"), (33, 64, 64, 16, 4, "none"),
    (1100, 128, 128, 16, 300, "each"), (2100, 64, 64, 8, 3, "requests"),
    # large adapters met by few rows (their sums come from a launch of their own), one and two tiles, the last group
    # of columns cut short
    (1, 2048, 1096, 64, 3, "one"), (20, 1544, 2056, 40, 6, "each"), (31, 512, 1600, 128, 2, "requests"),
]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,K,N,R,G,kind", SHAPES)
def test_lora_apply(dt, T, K, N, R, G, kind):
    x, A, B, scale, ad = lora_case(T, K, N, R, G, dt, T + K + N + R, kind)
    y = torch.randn(T, N, generator=gen(3)).to(dt)
    d, tol = lora_ref(x, A, B, scale, ad)
    l = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
    xc, ac, yc = x.cuda(), ad.cuda(), y.cuda()
    out = l.apply(xc, ac, yc, out=torch.empty_like(yc))
    close(out, y.double() + d, tol, "y")
    none = (ad < 0) | (ad >= G)
    assert same_bits(out.cpu()[none], y[none])
    same = l.apply(xc, ac, yc)  # in place
    assert same.data_ptr() == yc.data_ptr() and same_bits(same, out)
    zero = l.apply(xc, ac)  # no projection beside it
    close(zero, d, tol, "delta")
    assert (zero.cpu()[none] == 0).all()
    plain = tuning.LoRAAdapters(l.a, l.b).apply(xc, ac)  # scale 1
    d1, t1 = lora_ref(x, A, B, None, ad)
    close(plain, d1, t1, "delta without scale")


def test_lora_apply_rows_stay_apart():
    """NaN and infinities of one request, and of adapters that no row names,
    reach no other row; rows without an adapter keep their bits in place."""
    T, K, N, R, G = 70, 192, 136, 16, 6
    for dt in (BF16, F16, F32):
        x, A, B, scale, ad = lora_case(T, K, N, R, G, dt, 9, "each")
        ad[ad == 4] = 2
        ad[3], ad[8], ad[20], ad[21] = 1, 5, -7, G
        A[4], B[4] = float("nan"), float("nan")
        B[5, :, 3] = float("inf")
        ad[(ad == 5) & (torch.arange(T) != 8)] = 0
        x[3] = float("nan")
        ad[30] = -1
        x[30] = float("nan")
        y = torch.randn(T, N, generator=gen(1)).to(dt)
        y[30] = float("nan")
        y[31] = float("inf")
        out = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda()).apply(x.cuda(), ad.cuda(), y.cuda()).cpu()
        bad = torch.zeros(T, dtype=torch.bool)
        bad[[3, 8]] = True
        d, tol = lora_ref(torch.where(torch.isnan(x), 0, x), A.nan_to_num(0), B.nan_to_num(0, 0, 0), scale, ad)
        close(out[~bad], (y.double() + d)[~bad], tol[~bad], "other rows")
        none = (ad < 0) | (ad >= G)
        assert none[30] and same_bits(out[none], y[none])
        assert torch.isnan(out[3]).all() and not torch.isfinite(out[8]).any()


def test_lora_apply_large_and_small_values_f16():
    """f16 adapters whose inner sums lie outside f16's range."""
    T, K, N, R = 40, 1024, 64, 16
    for sx, sb in [(300.0, 2.0 ** -14), (2.0 ** -10, 8.0)]:
        x, A, B, _, ad = lora_case(T, K, N, R, 2, F16, 2, "one")
        x, A = (x.float() * sx).to(F16), (A.float() * (32 if sx > 1 else 2.0 ** -9)).to(F16)
        B = (torch.randn(2, N, R, generator=gen(4)) * sb).to(F16)
        scale = torch.tensor([1.0, 3.0])
        y = torch.zeros(T, N, dtype=F16)
        d, tol = lora_ref(x, A, B, scale, ad)
        out = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda()).apply(x.cuda(), ad.cuda(), y.cuda())
        keep = d.abs() < 60000
        assert keep.float().mean() > 0.9
        close(out.cpu()[keep], d[keep], tol[keep], "y")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,K,N,R,G,kind", SHAPES)
def test_lora_backward(dt, T, K, N, R, G, kind):
    x, A, B, scale, ad = lora_case(T, K, N, R, G, dt, T + K + N + R, kind)
    g = gen(8)
    dy, dx = (torch.randn(T, N, generator=g) * 0.5).to(dt), torch.randn(T, K, generator=g).to(dt)
    l = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
    ac = ad.cuda()
    gx, ga, gb = l.backward(x.cuda(), dy.cuda(), ac, dx=dx.cuda(), dx_out=torch.empty(T, K, dtype=dt, device="cuda"))
    rdx, rmag = dx.double().clone(), torch.zeros(T, K, dtype=torch.float64)
    ra, rb = torch.zeros(A.shape, dtype=torch.float64), torch.zeros(B.shape, dtype=torch.float64)
    ta, tb = ra.clone(), rb.clone()
    sp = split_err(dt)
    for a in range(G):
        r = (ad == a).nonzero()[:, 0]
        if not len(r):
            continue
        s, X, D, Aa, Bb = float(scale[a]), x[r].double(), dy[r].double(), A[a].double(), B[a].double()
        u, s1 = s * D @ Bb, s * X @ Aa.t()
        um, sm = s * D.abs() @ Bb.abs(), s * X.abs() @ Aa.abs().t()
        rdx[r] += u @ Aa
        rmag[r] = (um @ Aa.abs()) * ((N + R + 16) * U + sp)
        ra[a], ta[a] = u.t() @ X, (um.t() @ X.abs()) * ((N + len(r) + 16) * U + sp)
        rb[a], tb[a] = D.t() @ s1, (D.abs().t() @ sm) * ((K + len(r) + 16) * U + sp)
    close(gx, rdx, rmag, "dx")
    close(ga, ra, ta, "da")
    close(gb, rb, tb, "db")
    none = (ad < 0) | (ad >= G)
    assert same_bits(gx.cpu()[none], dx[none])
    # in place; without dx; the projection's gradient left out
    d2 = dx.cuda()
    hx, ha, hb = l.backward(x.cuda(), dy.cuda(), ac, dx=d2)
    assert hx.data_ptr() == d2.data_ptr() and same_bits(hx, gx) and same_bits(ha, ga) and same_bits(hb, gb)
    nx, na, nb = l.backward(x.cuda(), dy.cuda(), ac, need_dx=False)
    assert nx is None and same_bits(na, ga) and same_bits(nb, gb)
    zx = l.backward(x.cuda(), dy.cuda(), ac)[0]
    close(zx, rdx - dx.double(), rmag, "dx of the adapters alone")


@pytest.mark.parametrize("K,N,R", [(128, 264, 24), (2048, 2056, 64)])
def test_lora_backward_parts(K, N, R):
    """Each gradient asked for by itself through the C ABI has the bits of the
    call for all, and nothing else is written."""
    T, G = 29, 3
    x, A, B, scale, ad = lora_case(T, K, N, R, G, BF16, 4, "each")
    dy, dxi = torch.randn(T, N, generator=gen(1)).to(BF16), torch.randn(T, K, generator=gen(2)).to(BF16)
    xc, ac, dyc, dxc, a, b, s = (t.cuda() for t in (x, ad, dy, dxi, A, B, scale))
    want = tuning.LoRAAdapters(a, b, s).backward(xc, dyc, ac, dx=dxc, dx_out=torch.empty_like(dxc))
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    desc = _lib.Lora(a.data_ptr(), b.data_ptr(), s.data_ptr(), moe_dtype(BF16), R, N, K, G)
    need = lib.moe_lora_backward_workspace_bytes(C.byref(desc), T)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    for ask in [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)]:
        out = [torch.full_like(t, 9.0) for t in want]
        p = [o.data_ptr() if on else None for o, on in zip(out, ask)]
        ws.fill_(255)
        check(lib.moe_lora_backward(C.byref(desc), xc.data_ptr(), dyc.data_ptr(), T, ac.data_ptr(),
                                    dxc.data_ptr() if ask[0] else None, *p, ws.data_ptr(), need, st))
        torch.cuda.synchronize()
        for o, w, on in zip(out, want, ask):
            assert same_bits(o, w) if on else (o == 9).all(), ask
        assert (ws[need:] == 255).all()


@pytest.mark.parametrize("dt", [BF16, F32])
def test_lora_backward_many_rows(dt):
    """More rows than the first launch lists itself, spread unevenly over the
    adapters (one has none, one most of them), ids out of range among them."""
    T, K, N, R, G = 20011, 64, 40, 24, 70
    x, A, B, scale, _ = lora_case(T, K, N, R, G, dt, 5)
    g = gen(9)
    ad = torch.where(torch.rand(T, generator=g) < 0.6, 3, torch.randint(-1, G + 1, (T,), generator=g)).to(torch.int32)
    ad[ad == 5] = 6
    dy = torch.randn(T, N, generator=g).to(dt)
    gx, ga, gb = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda()).backward(x.cuda(), dy.cuda(), ad.cuda())
    sp = split_err(dt)
    assert (ga[5] == 0).all() and (gb[5] == 0).all()
    for a in (0, 3, 6, 63, 64, 69):
        r = (ad == a).nonzero()[:, 0]
        s, X, D, Aa, Bb = float(scale[a]), x[r].double(), dy[r].double(), A[a].double(), B[a].double()
        u, s1 = s * D @ Bb, s * X @ Aa.t()
        um, sm = s * D.abs() @ Bb.abs(), s * X.abs() @ Aa.abs().t()
        close(gx.cpu()[r], u @ Aa, (um @ Aa.abs()) * ((N + R + 16) * U + sp), f"dx {a}")
        close(ga[a], u.t() @ X, (um.t() @ X.abs()) * ((N + len(r) + 16) * U + sp), f"da {a}")
        close(gb[a], D.t() @ s1, (D.abs().t() @ sm) * ((K + len(r) + 16) * U + sp), f"db {a}")
    none = (ad < 0) | (ad >= G)
    assert (gx.cpu()[none] == 0).all()


@pytest.mark.parametrize("dt,T,K,N,R,G", [
    (BF16, 900, 2056, 136, 16, 120), (F16, 300, 1096, 520, 8, 200), (F32, 900, 136, 2056, 40, 120),
    (F32, 500, 1160, 264, 24, 250), (BF16, 700, 2824, 264, 40, 40), (F16, 1500, 520, 1928, 72, 50)])
def test_lora_backward_many_adapters(dt, T, K, N, R, G):
    """Few rows an adapter (blocks of the outer products take several column
    blocks) but for one that has half of all, and a few of about a dozen."""
    x, A, B, scale, _ = lora_case(T, K, N, R, G, dt, T + R)
    g = gen(T)
    ad = torch.randint(-1, G, (T,), generator=g)
    ad[torch.rand(T, generator=g) < 0.5] = 7
    ad[:60] = torch.arange(60) // 13 + 20
    ad[ad == 11] = 12
    ad = ad[torch.randperm(T, generator=g)].to(torch.int32)
    dy = torch.randn(T, N, generator=g).to(dt)
    l = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
    gx, ga, gb = (t.cpu() for t in l.backward(x.cuda(), dy.cuda(), ad.cuda()))
    sp = split_err(dt)
    for a in range(G):
        r = (ad == a).nonzero()[:, 0]
        if len(r) == 0:
            assert (ga[a] == 0).all() and (gb[a] == 0).all()
            continue
        s, X, D, Aa, Bb = float(scale[a]), x[r].double(), dy[r].double(), A[a].double(), B[a].double()
        u, s1 = s * D @ Bb, s * X @ Aa.t()
        um, sm = s * D.abs() @ Bb.abs(), s * X.abs() @ Aa.abs().t()
        close(gx[r], u @ Aa, (um @ Aa.abs()) * ((N + R + 16) * U + sp), f"dx {a}")
        close(ga[a], u.t() @ X, (um.t() @ X.abs()) * ((N + len(r) + 16) * U + sp), f"da {a}")
        close(gb[a], D.t() @ s1, (D.abs().t() @ sm) * ((K + len(r) + 16) * U + sp), f"db {a}")
    assert (gx[ad < 0] == 0).all()
    for first, again in zip((gx, ga, gb), l.backward(x.cuda(), dy.cuda(), ad.cuda())):
        assert same_bits(first, again.cpu())


def test_lora_backward_matches_differences():
    """Gradients against central differences of the float64 forward."""
    T, K, N, R, G = 12, 16, 24, 8, 3
    x, A, B, scale, ad = lora_case(T, K, N, R, G, F32, 5, "each", bstd=0.5)
    dy = torch.randn(T, N, generator=gen(6))
    gx, ga, gb = (t.double().cpu() for t in tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
                  .backward(x.cuda(), dy.cuda(), ad.cuda()))

    def loss(x, A, B):
        return (lora_ref(x, A, B, scale, ad)[0] * dy.double()).sum()

    h = 1e-3  # the loss is linear in each argument: differences have no truncation error
    at = [(0, (2, 3)), (0, (7, 15)), (1, (0, 1, 2)), (1, (2, 7, 9)), (2, (1, 20, 5)), (2, (0, 3, 0))]
    for which, i in at:
        v = [x.double(), A.double(), B.double()]
        up, dn = [t.clone() for t in v], [t.clone() for t in v]
        up[which][i] += h
        dn[which][i] -= h
        num = float((loss(*up) - loss(*dn)) / (2 * h))
        got = float((gx, ga, gb)[which][i])
        assert abs(num - got) <= 1e-9 + 200 * U * (1 + abs(num))


def test_lora_backward_rows_stay_apart():
    """NaN rows without an adapter or of another adapter leave the rest finite."""
    T, K, N, R, G = 50, 64, 72, 16, 4
    x, A, B, scale, ad = lora_case(T, K, N, R, G, BF16, 12, "each")
    dy = torch.randn(T, N, generator=gen(2)).to(BF16)
    ad[5], ad[6], ad[7] = -1, 2, G + 3
    x[5], x[7], dy[5], dy[7] = (float("nan"),) * 4
    x[6] = float("nan")
    l = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
    gx, ga, gb = l.backward(x.cuda(), dy.cuda(), ad.cuda())
    assert torch.isnan(ga[2]).all() and torch.isnan(gb[2]).all()
    rest = [0, 1, 3]
    assert torch.isfinite(ga[rest]).all() and torch.isfinite(gb[rest]).all() and torch.isfinite(gx).all()
    assert (gx[5] == 0).all() and (gx[7] == 0).all()


# ------------------------------------------------- streams, graphs, chains --

def tune_step(t):
    """A router with an adapter on it, tuned while the experts stay frozen:
    logits, routing, combine, losses, and all gradients back to the adapter."""
    lib, st = _lib.load(), C.c_void_p(torch.cuda.current_stream().cuda_stream)
    T, E, k, H, dt = t["T"], t["E"], t["k"], t["H"], moe_dtype(BF16)
    P = lambda v: C.c_void_p(v.data_ptr())  # noqa: E731
    e = lambda *s, d=torch.int32: torch.empty(*s, dtype=d, device="cuda")  # noqa: E731
    logits = e(T, E, d=BF16)
    check(lib.moe_router_logits(P(t["x"]), dt, T, H, P(t["W"]), dt, None, E, P(logits), st))
    t["lora"].apply(t["x"], t["ad"], logits)
    idx, w = e(T, k), e(T, k, d=F32)
    check(lib.moe_router_topk(P(logits), dt, T, E, k, 0, 1, None, P(idx), P(w), st))
    counts, offsets, perm, inv = e(E), e(E + 1), e(T * k), e(T * k)
    need = lib.moe_dispatch_workspace_bytes(T, k, E)
    ws = e(need, d=torch.uint8)
    check(lib.moe_dispatch_plan(P(idx), T, k, E, P(counts), P(offsets), P(perm), P(inv), P(ws), need, st))
    out = e(T, H, d=BF16)
    check(lib.moe_unpermute(P(t["Y"]), P(inv), P(w), T, H, k, P(out), dt, st))
    b = tuning.balance_loss(t["router"], logits, idx, mask=t["mask"])
    dY, dw = tuning.unpermute_backward(t["g"], t["Y"], inv, w)
    dl = tuning.router_backward(t["router"], logits, idx, dw, b.counts, 0.01, 0.001, mask=t["mask"])
    dx, da, db = t["lora"].backward(t["x"], dl, t["ad"])
    return dict(logits=logits, idx=idx, w=w, inv=inv, out=out, counts=b.counts, losses=b.losses, dY=dY, dw=dw, dl=dl,
                dx=dx, da=da, db=db, plan_counts=counts)


def tune_inputs(T=200, E=32, k=4, H=256, R=8, G=2):
    g = gen(21)
    x = torch.randn(T, H, generator=g).to(BF16).cuda()
    l = tuning.LoRAAdapters((torch.randn(G, R, H, generator=g) * H ** -0.5).to(BF16).cuda(),
                            (torch.randn(G, E, R, generator=g) * 0.1).to(BF16).cuda(), torch.tensor([1.0, 2.0]).cuda())
    return dict(T=T, E=E, k=k, H=H, x=x, W=(torch.randn(E, H, generator=g) * H ** -0.5).to(BF16).cuda(), lora=l,
                ad=(torch.arange(T) // 67 - 1).to(torch.int32).cuda(), Y=torch.randn(T * k, H, generator=g).to(BF16).cuda(),
                g=(torch.randn(T, H, generator=g) * 0.1).to(BF16).cuda(), router=MoERouter(E, k),
                mask=(torch.rand(T, generator=g) < 0.9).cuda())


def test_tuning_chain():
    """Forward and backward of a tuned router together: every stage against
    float64 on what the stage before it returned, and the whole chain's
    gradient against the whole loss."""
    t = tune_inputs()
    o = {k: v.cpu() for k, v in tune_step(t).items()}
    T, E, k, H, l = t["T"], t["E"], t["k"], t["H"], t["lora"]
    x, W, ad, m, g = t["x"].cpu(), t["W"].cpu(), t["ad"].cpu(), t["mask"].cpu(), t["g"].cpu()
    A, B, sc = l.a.cpu(), l.b.cpu(), l.scale.cpu()
    d, tol = lora_ref(x, A, B, sc, ad)
    base = x.double() @ W.double().t()
    mag = x.double().abs() @ W.double().abs().t()
    close(o["logits"], base + d, tol + mag * (H + 8) * U + base.abs() * 2.0 ** -8, "logits")
    counts, on = counts_of(o["idx"], m, E)
    assert torch.equal(o["counts"], counts)
    assert torch.equal(o["plan_counts"], counts_of(o["idx"], None, E)[0][:-1])
    r = t["router"]
    ref = router_ref(r, o["logits"], o["idx"], o["dw"], counts, 0.01, 0.001, m, None, None)
    close(o["dl"], ref, router_tol(r, o["logits"], o["idx"], o["dw"], counts, 0.01, 0.001, None, None), "d logits")
    # the whole loss, differentiated in float64 from the rows up; the bf16 roundings of logits, weights and d logits
    # on the way are what the stages' gradients carry: each term of da is off by a few 2^-8 of its magnitude
    A64, B64 = A.double().requires_grad_(True), B.double().requires_grad_(True)
    rows_y = torch.zeros(T, E, dtype=torch.float64)
    for a in range(2):
        at = (ad == a).nonzero()[:, 0]
        rows_y = rows_y.index_add(0, at, float(sc[a]) * (x[at].double() @ A64[a].t()) @ B64[a].t())
    s = base + rows_y
    w = weights64(s, o["idx"], r.gatingMode, True, None, 1.0, None)
    Y = t["Y"].cpu().double()[o["inv"].long()].view(T, k, H)
    on64 = on.double()[:, None]
    loss = ((w[..., None] * Y).sum(1) * g.double() * on64).sum()
    bal, z = losses64(s[on], counts[:-1], int(counts[-1]), k, SOFT)
    loss = loss + 0.01 * bal + 0.001 * z
    ga, gb = torch.autograd.grad(loss, [A64, B64])
    dlm = o["dl"].double().abs()
    for a in range(2):
        at = (ad == a).nonzero()[:, 0]
        um = float(sc[a]) * (dlm[at] + dlm[at].max(1, keepdim=True).values) @ B[a].double().abs()
        sm = float(sc[a]) * x[at].double().abs() @ A[a].double().abs().t()
        close(o["da"][a], ga[a], 4 * 2.0 ** -8 * um.t() @ x[at].double().abs(), f"da {a}")
        close(o["db"][a], gb[a], 4 * 2.0 ** -8 * (dlm[at] + dlm[at].max(1, keepdim=True).values).t() @ sm, f"db {a}")


def test_tuning_chain_repeats_and_streams():
    """The same bits from call to call, on another stream, and from two streams at once."""
    t = tune_inputs()
    want = {k: v.clone() for k, v in tune_step(t).items()}
    again = tune_step(t)
    assert all(same_bits(want[k], again[k]) for k in want)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    s1.wait_stream(torch.cuda.current_stream())
    s2.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        a = tune_step(t)
    with torch.cuda.stream(s2):
        b = tune_step(t)
    c = tuning.balance_loss(t["router"], want["logits"], want["idx"], mask=t["mask"], stream=s1)
    s1.synchronize()
    s2.synchronize()
    assert all(same_bits(want[k], a[k]) and same_bits(want[k], b[k]) for k in want)
    assert same_bits(c.losses, want["losses"])


def test_tuning_chain_in_two_graphs():
    """Two captured steps with inputs of their own, replayed in turn and between
    eager work, give the eager results every time."""
    t1, t2 = tune_inputs(), tune_inputs(T=90, E=16, k=2, H=128)
    want = [{k: v.clone() for k, v in tune_step(t).items()} for t in (t1, t2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in (t1, t2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(tune_step(t))
        graphs.append(gr)
    for rep in range(4):
        for i in (0, 1) if rep % 2 else (1, 0):
            for v in outs[i].values():
                v.zero_()
            graphs[i].replay()
            eager = tune_step((t1, t2)[1 - i])
            torch.cuda.synchronize()
            assert all(same_bits(want[i][k], outs[i][k]) for k in want[i]), f"replay {rep} of graph {i}"
            assert all(same_bits(want[1 - i][k], eager[k]) for k in eager)
    # new inputs in the same buffers
    t1["g"].mul_(2)
    new = {k: v.clone() for k, v in tune_step(t1).items()}
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(same_bits(new[k], outs[0][k]) for k in new) and not same_bits(new["da"], want[0]["da"])


def test_adapters_updated_and_moved():
    """A slot overwritten in place and tensors whose memory was exchanged are
    what the next call reads; memory of another shape or type is refused."""
    x, A, B, scale, ad = lora_case(6, 64, 64, 8, 2, BF16, 1, "one")
    a, b, s = A.cuda(), B.cuda(), scale.cuda()
    l = tuning.LoRAAdapters(a, b, s)
    xc, ac = x.cuda(), ad.cuda()
    l.apply(xc, ac)
    a[1].mul_(2)
    d, tol = lora_ref(x, a.cpu(), B, scale, ad)
    close(l.apply(xc, ac), d, tol, "slot overwritten")
    a.data, b.data, s.data = (A * 3).cuda(), (B * 2).cuda(), (scale + 1).cuda()
    d, tol = lora_ref(x, A * 3, B * 2, scale + 1, ad)
    close(l.apply(xc, ac), d, tol, "moved")
    a.data = a.data[:1]  # the same address, fewer adapters
    with pytest.raises(ValueError, match="b must be"):
        l.apply(xc, ac)
    a.data = A.cuda().half()
    with pytest.raises(ValueError, match="b dtype"):
        l.apply(xc, ac)


def test_refusals_on_the_gpu_launch_nothing():
    """A refused call leaves its outputs alone and the next one works."""
    x, A, B, scale, ad = lora_case(4, 64, 64, 8, 2, BF16, 1)
    l = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
    y = torch.full((4, 64), 3.0, dtype=BF16, device="cuda")
    with pytest.raises(_lib.MoeError, match="overlaps"):
        xc = x.cuda()
        l.apply(xc, ad.cuda(), out=xc)
    with pytest.raises(ValueError, match="on cpu"):
        l.apply(x.cuda(), ad, y)
    with pytest.raises(ValueError, match="contiguous"):
        l.apply(torch.zeros(64, 4, dtype=BF16, device="cuda").t(), ad.cuda(), y)
    torch.cuda.synchronize()
    assert (y == 3).all()
    l.apply(x.cuda(), ad.cuda(), y)
