"""Tuning and adapter entry points on the GPU at values of the far ends: infinities, inner sums outside a 16-bit type's
range, saturated sigmoids, rows of a type's lowest value. References and bounds in float64, as in test_gpu_tuning.py: a
result rounded to type t is off by eps(t)/2 of its value, a sum of n fp32 products by (n + c) 2^-24 of the sum of their
magnitudes, a factor kept as two 16-bit parts by 2^-17 of itself."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd.layer import MoEGatingMode, MoERouter  # noqa: E402

U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SOFT, PICK, SIGM = MoEGatingMode.softmaxThenTopK, MoEGatingMode.topKThenSoftmax, MoEGatingMode.sigmoidTopK
INF, NAN = float("inf"), float("nan")


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
    """|got - ref| <= half a step of got's type + tol where ref is finite; the same NaN and infinities elsewhere."""
    half = torch.finfo(got.dtype).eps / 2
    low = torch.finfo(got.dtype).smallest_normal * half
    got, ref, tol = got.double().cpu(), ref.double().cpu(), torch.as_tensor(tol, dtype=torch.float64)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), (
        f"{what}: {int((torch.isnan(got) & ~torch.isnan(ref)).sum())} NaN too many, "
        f"{int((~torch.isnan(got) & torch.isnan(ref)).sum())} too few")
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities"
    bound = half * (ref.abs() + tol) + tol + low + torch.finfo(torch.float32).tiny
    bad = ((got - ref).abs() > bound) & fin
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{((got - ref).abs() / bound)[fin].max():.3g} of the bound")


# ------------------------------------------------------------- infinities --

def products(a, b):
    """Rows of a against rows of b in float64, every product and sum as IEEE has it."""
    return (a[:, None, :] * b[None, :, :]).sum(-1)


def adapter_case(T, K, N, R, G, dt, seed):
    """Signed inputs whose inner sums are far from zero (1 to 2 of one sign or the other): their signs are not in doubt."""
    g = gen(seed)
    x = (torch.rand(T, K, generator=g) + 0.5).to(dt)
    sign = torch.where(torch.rand(G, R, generator=g) < 0.5, -1.0, 1.0)
    A = (sign[:, :, None] * (torch.rand(G, R, K, generator=g) + 0.5) * 1.5 / K).to(dt)
    B = ((torch.rand(G, N, R, generator=g) + 0.1) * torch.where(torch.rand(G, N, 1, generator=g) < 0.5, -0.1, 0.1)).to(dt)
    dy = (torch.rand(T, N, generator=g) + 0.5).to(dt)
    return x, A, B, torch.rand(G, generator=g) + 0.5, torch.randint(-1, G, (T,), generator=g).to(torch.int32), dy


def adapter_ref(x, A, B, scale, ad, dy):
    """y, dx, dA, dB of the adapters in float64, with bounds on finite values' fp32 errors."""
    T, K, N, R = x.shape[0], x.shape[1], B.shape[1], A.shape[1]
    sp = 0.0 if x.dtype == F32 else 2.0 ** -17
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    y, dx, dA, dB = z(T, N), z(T, K), z(*A.shape), z(*B.shape)
    ty, tx, tA, tB = z(T, N), z(T, K), z(*A.shape), z(*B.shape)
    for a in range(A.shape[0]):
        r = (ad == a).nonzero()[:, 0]
        if not len(r):
            continue
        s, X, D, Aa, Bb = float(scale[a]), x[r].double(), dy[r].double(), A[a].double(), B[a].double()
        si, u = s * products(X, Aa), s * products(D, Bb.t())
        sm, um = s * products(X.abs(), Aa.abs()), s * products(D.abs(), Bb.abs().t())
        y[r], ty[r] = products(si, Bb), products(sm, Bb.abs()) * ((K + R + 16) * U + sp)
        dx[r], tx[r] = products(u, Aa.t()), products(um, Aa.abs().t()) * ((N + R + 16) * U + sp)
        dA[a], tA[a] = products(u.t(), X.t()), products(um.t(), X.abs().t()) * ((N + len(r) + 16) * U + sp)
        dB[a], tB[a] = products(D.t(), si.t()), products(D.abs().t(), sm.t()) * ((K + len(r) + 16) * U + sp)
    return (y, dx, dA, dB), (ty, tx, tA, tB)


# ranks that fill a product's inner axis and ranks that do not; one and several steps; few rows that large adapters meet
# in two launches; one adapter met by all rows
ADAPTERS = [(40, 72, 136, 8, 2), (33, 64, 200, 16, 3), (70, 136, 72, 24, 2), (50, 64, 64, 32, 1), (150, 72, 264, 40, 2),
            (64, 64, 136, 64, 2), (90, 72, 72, 72, 1), (35, 64, 136, 128, 2), (3, 1032, 1096, 64, 2)]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,K,N,R,G", ADAPTERS)
@pytest.mark.parametrize("where", ["a", "b", "x", "dy", "xb", "none"])
def test_adapters_carry_infinities(dt, T, K, N, R, G, where):
    """An infinity in a factor is an infinity (or NaN where it meets a zero or its opposite) in the sums that have it, and
    leaves all others as they are."""
    x, A, B, scale, ad, dy = adapter_case(T, K, N, R, G, dt, T + R)
    ad[0], ad[-1] = 0, G - 1
    if where == "a":
        A[0, R - 1, 3], A[G - 1, 0, K - 1] = INF, -INF
    if where in ("b", "xb"):
        B[0, 5, R - 1], B[0, N - 1, 0], B[G - 1, 7, R // 2] = INF, -INF, INF
        B[0, 9, 1], B[0, 9, 2] = INF, 0.0
    if where in ("x", "xb"):
        x[0, 2], x[-1, K - 1] = INF, -INF
    if where == "dy":
        dy[0, 4], dy[-1, N - 1] = INF, -INF
    l = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
    (y, dx, dA, dB), (ty, tx, tA, tB) = adapter_ref(x, A, B, scale, ad, dy)
    if where != "none":
        assert torch.isinf(torch.cat([t.flatten() for t in (y, dx, dA, dB)])).any()
    close(l.apply(x.cuda(), ad.cuda()), y, ty, "y")
    gx, ga, gb = l.backward(x.cuda(), dy.cuda(), ad.cuda())
    close(gx, dx, tx, "dx")
    close(ga, dA, tA, "da")
    close(gb, dB, tB, "db")


@pytest.mark.parametrize("T,R", [(40, 16), (40, 24), (100, 64), (100, 128)])
def test_f16_sums_beside_an_infinite_one(T, R):
    """f16 inner sums outside f16's range keep their bits in a row, and in steps of a gradient, that hold an infinite one."""
    K, N, G = 64, 72, 1
    x, A, B, scale, ad, dy = adapter_case(T, K, N, R, G, F16, R)
    ad.fill_(0)
    A, B, dy = A * 0 + 1000, B * 0 + 2.0 ** -10, dy * 2.0 ** -11
    A[0, 1:R:2] = 2.0 ** -9  # small sums beside the large ones
    A[0, R - 1, 3] = INF
    x = x * 4
    B[0, :, R - 1] = 0  # (the infinite sum times zero: y is NaN, the gradients of the other ranks are not)
    l = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
    (_, dx, dA, dB), (_, tx, tA, tB) = adapter_ref(x, A, B, scale, ad, dy)
    assert float((x[0].float() @ A[0, 0].float()) * scale[0]) > 65504 and torch.isfinite(dB[0, :, :R - 1]).all()
    assert dB[0, :, :R - 1].max() < 65504
    y = l.apply(x.cuda(), ad.cuda())
    assert torch.isnan(y).all()
    gx, ga, gb = l.backward(x.cuda(), dy.cuda(), ad.cuda())
    close(gx, dx, tx, "dx")
    close(ga, dA, tA, "da")
    close(gb, dB, tB, "db")


@pytest.mark.parametrize("R", [16, 24, 64])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_inner_sums_of_many_sizes(dt, R):
    """Sums from the largest to 2^-20 of it, weighed so that each matters: as two 16-bit parts they keep 2^-17 (bf16), or
    2^-23 of themselves and 2^-39 of the largest (f16)."""
    T, K, N = 40, 64, 72
    g = gen(R)
    x = torch.randn(T, K, generator=g).to(dt)
    size = 2.0 ** -(torch.arange(R) % 21).float()
    A = (torch.randn(1, R, K, generator=g) * 64 * size[:, None]).to(dt)
    B = (torch.randn(1, N, R, generator=g) * 2.0 ** -14 / size).to(dt)
    dy = (torch.randn(T, N, generator=g) * 2.0 ** -8).to(dt)
    ad = torch.zeros(T, dtype=torch.int32)
    X, D, Aa, Bb = x.double(), dy.double(), A[0].double(), B[0].double()
    s, sm, u, um = X @ Aa.t(), X.abs() @ Aa.abs().t(), D @ Bb, D.abs() @ Bb.abs()

    def parts(v, over):  # what two parts may leave out
        return v.abs() * 2.0 ** -17 if dt == BF16 else v.abs() * 2.0 ** -23 + 2.0 ** -39 * v.abs().amax(over, keepdim=True)

    l = tuning.LoRAAdapters(A.cuda(), B.cuda())
    close(l.apply(x.cuda(), ad.cuda()), s @ Bb.t(), parts(s, 1) @ Bb.abs().t() + (sm @ Bb.abs().t()) * (K + R + 16) * U, "y")
    gx, ga, gb = l.backward(x.cuda(), dy.cuda(), ad.cuda())
    close(gx, u @ Aa, parts(u, 1) @ Aa.abs() + (um @ Aa.abs()) * (N + R + 16) * U, "dx")
    whole = R > 16  # else the gradients take the sums as they are
    close(ga[0], u.t() @ X, whole * parts(u, (0, 1)).t() @ X.abs() + (um.t() @ X.abs()) * (N + T + 16) * U, "da")
    close(gb[0], D.t() @ s, whole * D.abs().t() @ parts(s, (0, 1)) + (D.abs().t() @ sm) * (K + T + 16) * U, "db")


# ---------------------------------------------------------------- routers --

def case(T, E, k, seed, lo, hi):
    g = gen(seed)
    logits = torch.rand(T, E, generator=g) * (hi - lo) + lo
    idx = torch.rand(T, E, generator=g).topk(k).indices.to(torch.int32)
    counts = torch.cat([torch.bincount(idx.flatten().long(), minlength=E), torch.tensor([T])]).to(torch.int32)
    return logits, idx, counts


@pytest.mark.parametrize("lo,hi,deep", [(10.0, 20.0, None), (15.0, 80.0, None), (-80.0, -10.0, None), (-2.0, 2.0, None),
                                        (-2.0, 2.0, -200.0), (-2.0, 2.0, -INF), (-2.0, 2.0, INF)])
@pytest.mark.parametrize("norm", [False, True])
def test_saturated_sigmoids_keep_their_slope(lo, hi, deep, norm):
    """v (1 - v) is not rounded away where v is near 1: the gradients are right relative to the slope, not only to 1."""
    T, E, k = 50, 24, 5
    lg, idx, counts = case(T, E, k, 3, lo, hi)
    if deep is not None:  # every third expert: its slope is 0 in fp32
        lg[:, ::3] = deep
    dw = torch.randn(T, k, generator=gen(4))
    s, at = lg.double(), idx.long()
    v, slope = torch.sigmoid(s), torch.sigmoid(s) * torch.sigmoid(-s)
    # the slope: the exponential (2 ulp of the hardware's power and its correction), a sum, a reciprocal and two products
    c = 12 * U
    # the weights' gradient: g, or (g - sum g w / S) / S, times the slope of the pick
    g, w = dw.double(), v.gather(1, at)
    mag = g.abs()
    if norm:
        S = w.sum(1, keepdim=True) + 1e-20
        Gn = (g * w).sum(1, keepdim=True) / S
        mag = (g.abs() + (g.abs() * w).sum(1, keepdim=True) / S) / S
        g = (g - Gn) / S
    want = torch.zeros(T, E, dtype=torch.float64).scatter_add(1, at, g * slope.gather(1, at))
    tol = torch.zeros(T, E, dtype=torch.float64).scatter_add(1, at, mag * slope.gather(1, at)) * (c + (2 * k + 16) * U)
    r = MoERouter(E, k, SIGM, norm)
    got = tuning.router_backward(r, lg.cuda(), idx.cuda(), dw.cuda())
    close(got, want, tol, "weights")
    # the balance loss: q (1 - v) (f - sum f q), q = v / sum v
    f = 0.5 * E * counts[:-1].double() / (k * T * T)
    q = v / v.sum(1, keepdim=True)
    mean = (f * q).sum(1, keepdim=True)
    want = q * torch.sigmoid(-s) * (f - mean)
    tol = q * torch.sigmoid(-s) * (f + mean) * (c + (2 * E + 16) * U)
    got = tuning.router_backward(r, lg.cuda(), idx.cuda(), counts=counts.cuda(), balance_coef=0.5)
    close(got, want, tol, "balance")


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("gating,norm", [(PICK, True), (SOFT, True), (SIGM, False), (SIGM, True)])
def test_weights_gradient_beside_infinite_logits(dt, gating, norm):
    """Where the weights are functions of the picks alone, what the other experts hold is not in their gradient."""
    T, E, k = 21, 40, 4
    lg, idx, _ = case(T, E, k, 5, -2.0, 2.0)
    lg, at = lg.to(dt), idx.long()
    dw = torch.randn(T, k, generator=gen(6))
    l = lg.double().gather(1, at).requires_grad_(True)
    w = torch.softmax(l, 1) if gating != SIGM else torch.sigmoid(l)
    scale = 1.0
    if gating == SIGM and norm:
        scale = 1.0 / w.detach().sum(1, keepdim=True)
        w = w / w.sum(1, keepdim=True)
    g = torch.autograd.grad((w * dw.double()).sum(), l)[0]
    want = torch.zeros(T, E, dtype=torch.float64).scatter(1, at, g)
    other = torch.ones(T, E, dtype=torch.bool).scatter(1, at, False)
    far = torch.tensor([INF, NAN, -INF])[torch.randint(0, 3, (T, E), generator=gen(7))].to(dt)
    lg = torch.where(other & (torch.rand(T, E, generator=gen(8)) < 0.2), far, lg)
    tol = (2 * dw.double().abs().sum(1, keepdim=True) * scale * (k + 24) * U).expand(T, E)
    close(tuning.router_backward(MoERouter(E, k, gating, norm), lg.cuda(), idx.cuda(), dw.cuda()), want, tol, "d logits")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("gating,norm,bias", [(SOFT, True, False), (SOFT, False, False), (SOFT, True, True), (PICK, True, False)])
def test_rows_of_far_values(dt, gating, norm, bias):
    """Rows that a mask filled with the type's lowest value, wholly or but for a few, and rows far from zero: softmax only
    depends on the distance to the row's maximum."""
    T, E, k = 12, 20, 3
    lg, idx, counts = case(T, E, k, 7, -1.0, 1.0)
    low, high = torch.finfo(dt).min, torch.finfo(dt).max
    lg[0] = low
    lg[1], lg[1, 4], lg[1, 11] = low, 0.5, -0.25
    lg[2], lg[2, 3] = low, high
    lg[3] = high
    for t, far in ((4, 1e5), (5, 3e9), (6, -3e10), (7, 1e20), (8, 2.0 ** 22)):
        lg[t] = lg[t] * 4 + far
    lg[9] = torch.where(torch.arange(E) % 2 == 0, 2.0 ** 21, 2.0 ** 21 + 1)
    lg = lg.clamp(low, high).to(dt)
    eb = torch.full((E,), 0.125) if bias else None
    r = MoERouter(E, k, gating, norm, cuda(eb))
    s, at = lg.double(), idx.long()
    p = torch.softmax(s, 1)
    c = (E + 16) * U
    b = tuning.balance_loss(r, lg.cuda(), idx.cuda())
    close(b.prob_sum, p.sum(0), p.sum(0) * (c + (T + 8) * U), "P")
    bal = E * (counts[:-1].double() / (k * T) * p.sum(0) / T).sum()
    lse = torch.logsumexp(s, 1)
    z = lse.square().sum() / T  # past fp32's range with the largest values of bf16 and fp32
    z = torch.where(z > torch.finfo(F32).max, INF, z)
    close(b.losses, torch.stack([bal, z]), torch.stack([bal * (c + (T + 8) * U), z * (c + (T + 8) * U)]).nan_to_num(0, 0), "losses")
    dw = torch.randn(T, k, generator=gen(2))
    l = lg.double().requires_grad_(True)
    q, g = torch.softmax(l, 1), dw.double()
    if gating == PICK or (norm and eb is None):
        w = torch.softmax(l.gather(1, at), 1)
        scale = 1.0
    else:
        w = q.gather(1, at) + (0.0 if eb is None else 0.125)
        scale = torch.ones(T, 1)
        if norm:
            scale = 2.0 / w.detach().sum(1, keepdim=True)
            w = w / w.sum(1, keepdim=True)
    loss = (w * g).sum() + 0.5 * E * (counts[:-1].double() / (k * T) * q.sum(0) / T).sum()
    want = torch.autograd.grad(loss, l)[0]
    tol = ((2 * g.abs().sum(1, keepdim=True) * scale + E * counts[:-1].max() / (k * T * T)) * (E + k + 24) * U).expand(T, E)
    got = tuning.router_backward(r, lg.cuda(), idx.cuda(), dw.cuda(), counts.cuda(), 0.5)
    close(got, want, tol, "d logits")


@pytest.mark.parametrize("T", [30, 4000])
def test_sigmoid_router_with_infinite_logits(T):
    """sigmoid(inf) is 1 and sigmoid(-inf) 0: the probabilities and the balance loss stay finite, and z does not."""
    E, k = 16, 3
    lg, idx, counts = case(T, E, k, 9, -2.0, 2.0)
    lg[2, 5], lg[3, 1], lg[4, :8], lg[5] = INF, -INF, INF, -INF
    r = MoERouter(E, k, SIGM)
    b = tuning.balance_loss(r, lg.cuda(), idx.cuda())
    v = torch.sigmoid(lg.double())
    P = torch.where(v.sum(1, keepdim=True) > 0, v / v.sum(1, keepdim=True), 0.0).sum(0)  # row 5: no probability
    c = (E + 16 + T + 8) * U
    close(b.prob_sum, P, P * c, "P")
    bal = E * (counts[:-1].double() / (k * T) * P / T).sum()
    close(b.losses[:1], bal[None], bal * c, "balance")
    assert torch.isnan(b.losses[1])
    lg[7, 2] = NAN
    b = tuning.balance_loss(r, lg.cuda(), idx.cuda())
    assert torch.isnan(b.losses).all() and torch.isnan(b.prob_sum).all()
