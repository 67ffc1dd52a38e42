"""Gradients through frozen quantised experts on the GPU against float64
restatements.

Tolerances follow from the arithmetic: a result rounded to type t is off by at
most eps(t)/2 of its value, a sum of n fp32 products by at most (n + c) 2^-24 of
the sum of their magnitudes, and a weight that enters a product in type t by
eps(t)/2 of itself (f16 below 2^-14: 2^-25)."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_tuning import BF16, F16, F32, U, close, cuda, gen, same_bits  # noqa: E402

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd._lib import MoeError, check  # noqa: E402
from ffai_amd.layer import StackedExperts, moe_dtype  # noqa: E402

SWIGLU, GPTOSS, GEGLU, RELU2 = _lib.MOE_ACT_SWIGLU, _lib.MOE_ACT_GPTOSS, _lib.MOE_ACT_GEGLU, _lib.MOE_ACT_RELU2
ALPHA, LIMIT = 1.702, 7.0


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    _lib.load()
    yield
    torch.cuda.synchronize()


def half(t):
    return torch.finfo(t).eps / 2


# --------------------------------------------------------------- products --

def stack(E, N, K, bits, gs, sb, seed):
    """A quantised stack on the host and its weights in float64."""
    g = gen(seed)
    q = torch.randint(0, 2 ** bits, (E, N, K), generator=g)
    s = (torch.rand(E, N, K // gs, generator=g) + 0.5).mul_(0.2 / 2 ** bits).to(sb)
    b = (-s.float() * (2 ** bits - 1) / 2 + torch.randn(E, N, K // gs, generator=g) * 0.01).to(sb)
    bit = (q[..., None] >> torch.arange(bits)) & 1
    words = bit.reshape(E, N, K * bits // 32, 32) << torch.arange(32)
    w = words.sum(-1)
    w = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    W = q.double() * s.double().repeat_interleave(gs, 2) + b.double().repeat_interleave(gs, 2)
    return StackedExperts(w.cuda(), s.cuda(), b.cuda(), bits, gs), W


def plan(idx, E):
    """perm, inv_perm, offsets of picks idx [T, k]; an id outside has no position."""
    flat = idx.flatten().long()
    on = (flat >= 0) & (flat < E)
    order = torch.where(on, flat, E).argsort(stable=True)
    inv = torch.full((flat.numel(),), -1, dtype=torch.int32)
    used = int(on.sum())
    inv[order[:used]] = torch.arange(used, dtype=torch.int32)
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = torch.bincount(flat[on], minlength=E).cumsum(0)
    return order.to(torch.int32), inv.reshape(idx.shape), offsets


def picks(T, E, k, seed, kind="even"):
    g = gen(seed)
    score = torch.rand(T, E, generator=g)
    if kind == "one":  # everybody's first pick is expert 0, the last experts have no rows
        score[:, 0] += 2
        score[:, E // 2:] -= 2
    idx = score.topk(k).indices.to(torch.int32)
    if kind == "steep":  # from no row to several hundred
        idx = (torch.rand(T, k, generator=g) ** 3 * E).long().clamp(max=E - 1).to(torch.int32)
    if kind == "some":  # picks of no expert
        idx = torch.where(torch.rand(T, k, generator=g) < 0.2, torch.full_like(idx, -1), idx)
    return idx


def grad64(Ws, dys, offsets, perm, top_k, base):
    """(gradient, sum of magnitudes, of dy alone) in float64."""
    M, K = base.shape
    out, mag, only = base.double().clone(), torch.zeros(M, K, dtype=torch.float64), torch.zeros(M, 1, dtype=torch.float64)
    rows = torch.arange(M) if perm is None else perm.long() // top_k
    for W, dy in zip(Ws, dys):
        for e in range(W.shape[0]):
            a, b = int(offsets[e]), int(offsets[e + 1])
            d = dy[rows[a:b]].double()
            out[a:b] += d @ W[e]
            mag[a:b] += d.abs() @ W[e].abs()
            only[a:b] += d.abs().sum(1, keepdim=True)
    return out, mag, only


def product_tol(dt, mag, only, n, base):
    wt = {F32: 0.0, F16: half(F16), BF16: half(BF16)}[dt]
    tiny = 2.0 ** -25 if dt == F16 else 0.0
    return mag * (wt * (1 + n * U) + (n + 8) * U) + only * tiny + base.double().abs() * 2 * U


CASES = [
    # T, E, k, N, K, bits, gs, pair, gather, add, kind
    (1, 4, 1, 64, 64, 4, 64, False, False, False, "even"), (1, 8, 2, 104, 96, 4, 32, True, False, False, "even"),
    (1, 3, 3, 8, 32, 8, 32, False, True, True, "even"), (5, 60, 4, 72, 160, 5, 32, False, True, False, "even"),
    (37, 16, 4, 200, 192, 3, 64, True, False, True, "even"), (37, 16, 4, 256, 256, 6, 64, False, True, False, "one"),
    (64, 8, 2, 128, 320, 2, 32, True, False, False, "some"), (333, 8, 2, 96, 384, 4, 128, False, False, True, "one"),
    (700, 2, 1, 40, 288, 4, 32, True, False, False, "one"), (513, 1, 1, 136, 544, 8, 32, False, True, False, "even"),
    (129, 200, 3, 64, 128, 4, 64, False, False, False, "some"), (300, 4, 2, 520, 640, 3, 128, False, True, True, "even"),
    # the kernels of many and of few rows: shapes of tiles from 32 to 256 rows, blocks of 128 and 256 columns
    (4000, 32, 1, 40, 2048, 4, 64, False, True, False, "steep"), (3000, 32, 1, 104, 1952, 3, 32, True, False, True, "steep"),
    (2600, 64, 1, 72, 1184, 8, 32, False, False, False, "steep"), (1100, 33, 1, 136, 2080, 6, 32, True, False, False, "one"),
    (300, 300, 2, 40, 512, 4, 64, True, False, False, "steep"), (500, 1024, 2, 72, 224, 5, 32, False, True, True, "steep"),
    (600, 1024, 1, 8, 32, 2, 32, False, False, False, "one"), (1, 1024, 3, 264, 288, 8, 32, False, True, False, "even"),
    (150, 3, 2, 1032, 96, 6, 32, True, False, False, "even"), (90, 5, 2, 48, 1056, 5, 32, True, True, True, "even"),
]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,E,k,N,K,bits,gs,pair,gather,add,kind", CASES)
def test_expert_matmul_backward(dt, T, E, k, N, K, bits, gs, pair, gather, add, kind):
    M, g = T * k, gen(T + N)
    sb = dt if dt == F32 or T != 37 else (F16 if dt == BF16 else BF16)  # (scales of the other 16-bit type too)
    stacks = [stack(E, N, K, bits, gs, sb, 7 * i + E) for i in range(2 if pair else 1)]
    perm, _, offsets = plan(picks(T, E, k, T, kind), E)
    if not gather:
        perm = None
    dys = [(torch.randn(T if gather else M, N, generator=g) * 0.01).to(dt) for _ in stacks]
    base = (torch.randn(M, K, generator=g) * 0.01).to(dt) if add else torch.zeros(M, K, dtype=dt)
    ref, mag, only = grad64([w for _, w in stacks], dys, offsets, perm, k, base)
    mark = torch.full((M, K), 7.25, dtype=dt)
    kw = dict(perm=cuda(perm), top_k=k, dx=base.cuda() if add else None, out=mark.cuda())
    if pair:
        kw.update(proj2=stacks[1][0], dy2=dys[1].cuda())
    got = tuning.expert_matmul_backward(stacks[0][0], dys[0].cuda(), offsets.cuda(), **kw)
    used = int(offsets[-1])
    n = N * len(stacks)
    close(got[:used], ref[:used], product_tol(dt, mag, only, n, base)[:used], "dx")
    assert (got[used:] == 7.25).all(), "rows behind the last expert's were written"
    if add:  # into the gradient itself, and the same bits again
        kw["out"] = None
        again = tuning.expert_matmul_backward(stacks[0][0], dys[0].cuda(), offsets.cuda(), **kw)
        assert again is kw["dx"] and same_bits(again[:used], got[:used]) and same_bits(again[used:].cpu(), base[used:])


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_expert_matmul_backward_keeps_rows_apart(dt):
    """An infinity or a NaN stays in its own row of dy, and in its own expert."""
    T, E, N, K = 300, 4, 64, 128
    p, _ = stack(E, N, K, 4, 64, dt, 3)
    perm, _, offsets = plan(picks(T, E, 1, 5), E)
    dy = (torch.randn(T, N, generator=gen(1)) * 0.01).to(dt)
    plain = tuning.expert_matmul_backward(p, dy.cuda(), offsets.cuda())
    bad = dy.clone()
    bad[17, 5], bad[200, 63] = float("nan"), float("inf")
    got = tuning.expert_matmul_backward(p, bad.cuda(), offsets.cuda())
    keep = torch.ones(T, dtype=torch.bool)
    keep[[17, 200]] = False
    assert same_bits(got[keep.cuda()], plain[keep.cuda()])
    assert got[17].isnan().all() and not got[200].isfinite().any()
    p.scales[2, 9, 0] = float("nan")
    got = tuning.expert_matmul_backward(p, dy.cuda(), offsets.cuda())
    a, b = int(offsets[2]), int(offsets[3])
    assert got[a:b, :64].isnan().all() and same_bits(got[a:b, 64:], plain[a:b, 64:])
    assert same_bits(got[:a], plain[:a]) and same_bits(got[b:], plain[b:])


def test_expert_matmul_backward_small_gradients():
    """bfloat16 gradients far below f16's range keep their precision."""
    T, E, N, K = 70, 2, 128, 128
    p, W = stack(E, N, K, 4, 64, BF16, 3)
    _, _, offsets = plan(picks(T, E, 1, 5), E)
    dy = (torch.randn(T, N, generator=gen(1)) * torch.logspace(-30, 30, T)[:, None]).to(BF16)
    zero = torch.zeros(T, K, dtype=BF16)
    ref, mag, only = grad64([W], [dy], offsets, None, 1, zero)
    close(tuning.expert_matmul_backward(p, dy.cuda(), offsets.cuda()), ref, product_tol(BF16, mag, only, N, zero), "dx")


# ------------------------------------------------------------- activation --

def kept64(v):
    """codes and exponent bytes of the definition, by exact arithmetic."""
    blocks = v.double().reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    top = blocks.abs().amax(-1)
    e = torch.zeros(top.shape, dtype=torch.int64)
    for c in range(8, -1, -1):  # the least e with top < 127.5 * 2^(e - 133)
        low = e + 2 ** c - 1
        e = torch.where(top >= 127.5 * torch.exp2((low - 133).double()), low + 1, e)
    e = torch.where(torch.isfinite(top), e.clamp(max=255), torch.full_like(e, 255))
    codes = torch.round(blocks * torch.exp2((133 - e).double())[..., None])
    codes = torch.where((e == 255)[..., None], torch.zeros_like(codes), codes)
    return codes.reshape(v.shape).to(torch.int8), e.to(torch.uint8)


def values64(codes, e):
    step = torch.exp2(e.double() - 133)
    step = torch.where(e == 255, torch.full_like(step, float("nan")), step)
    return codes.double() * step.repeat_interleave(32, -1)


def act64(act, g, u, dt):
    """(value, slope in g, slope in u) in float64; gelu's value rounded to dt."""
    if act == RELU2:
        r = u.clamp(min=0)
        return r * r, None, 2 * r
    if act == GPTOSS:
        gc, uc = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        s = torch.sigmoid(ALPHA * gc)
        a = gc * s
        return a * (uc + 1), torch.where(g > LIMIT, 0.0, (s + ALPHA * a * (1 - s)) * (uc + 1)), torch.where(u.abs() > LIMIT, 0.0, a)
    if act == GEGLU:
        c = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * c * (g + 0.044715 * g ** 3))
        d = s + g * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * g * g)
        return g * s * u, d * u, g * s
    s = torch.sigmoid(g)
    return g * s * u, (s + g * s * (1 - s)) * u, g * s


# The logistic's exponent is a product rounded in fp32 (|x| 2^-24 of it, and so
# of the exponential), its exponential, sum and reciprocal are 4 roundings more;
# a slope adds terms of up to (1 + |a g|) of the value's size.
def act_tol(act, g, u, dt):
    x = (u if g is None else g).abs().clamp(max=100.0)
    c = 16 * U * (1 + 2 * x) * (1 + 2 * x)
    big = (x + 1) * (u.abs().clamp(max=8.0 if act == GPTOSS else 1e30) + 1) if act != RELU2 else (x + 1) ** 2
    gelu = half(dt) * x * u.abs() if act == GEGLU else 0.0
    return c * big + gelu, c * big, c * (x + 1) + (half(dt) * x if act == GEGLU else 0.0)


def projections(act, M, n, dt, seed):
    g = gen(seed)
    v = torch.randn(1 if act == RELU2 else 2, M, n, generator=g) * 1.5
    v = v * torch.exp(torch.randn(1, 1, n, generator=g) * 0.8)
    return v.to(dt)


SHAPES = [(1, 32), (3, 96), (37, 64), (130, 512), (64, 768), (17, 2880), (5, 4128)]


@pytest.mark.parametrize("act", [SWIGLU, GPTOSS, GEGLU, RELU2])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("M,n", SHAPES)
def test_activation_save(act, dt, M, n):
    v = projections(act, M, n, dt, M + n)
    gate = None if act == RELU2 else v[0].cuda()
    h, kept = tuning.activation_save(gate, v[-1].cuda(), act, ALPHA, LIMIT)
    codes, e = kept64(v)
    assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), e)
    # what was kept is off by at most half a step
    step = torch.exp2(e.double() - 133).repeat_interleave(32, -1)
    assert ((values64(codes, e) - v.double()).abs() <= step / 2).all()
    same = torch.empty_like(h)
    check(_lib.load().moe_activation_apply(None if gate is None else gate.data_ptr(), v[-1].cuda().data_ptr(), same.data_ptr(),
                                           M * n, moe_dtype(dt), act, ALPHA, LIMIT, torch.cuda.current_stream().cuda_stream))
    assert same_bits(h, same)
    for to in (BF16, F16, F32):
        ref = values64(codes, e).to(to)
        assert torch.equal(kept.restore(to).cpu(), ref)


def test_activation_save_extremes():
    """Zeros, the smallest and largest values, edges of a step, infinities, NaN."""
    v = torch.zeros(1, 16, 32)
    v[0, 1, 3] = 1e-45
    v[0, 2, 5], v[0, 2, 6] = 2.0 ** -126, -2.0 ** -127
    v[0, 3, :] = 127.5 * 2.0 ** -6
    v[0, 4, :] = torch.nextafter(torch.tensor(127.5 * 2.0 ** -6), torch.tensor(0.0))
    v[0, 5, 0], v[0, 5, 1] = 3.3e38, 1.0
    v[0, 6, 0] = torch.finfo(torch.float32).max
    v[0, 7, 9] = float("inf")
    v[0, 8, 31] = float("nan")
    v[0, 9, 0], v[0, 9, 1], v[0, 9, 2] = 1.0, 0.5 * 2.0 ** -6, 1.5 * 2.0 ** -6  # ties go to the even code
    v[0, 10, :] = -0.0
    v[0, 11, 2], v[0, 11, 3] = 2.0 ** -120, 2.0 ** -127
    _, kept = tuning.activation_save(None, v[0].cuda(), RELU2)
    codes, e = kept64(v)
    assert torch.equal(kept.scales.cpu(), e) and torch.equal(kept.codes.cpu(), codes)
    back = kept.restore(torch.float32).cpu()
    assert back[0, 6:9].isnan().all() and torch.equal(back[0, :6].double(), values64(codes, e)[0, :6])


@pytest.mark.parametrize("act", [SWIGLU, GPTOSS, GEGLU, RELU2])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("M,n", SHAPES)
def test_activation_backward(act, dt, M, n):
    codes, e = kept64(projections(act, M, n, dt, M * n))
    v, g = values64(codes, e), gen(n)
    dh = (torch.randn(M, n, generator=g) * 0.01).to(dt)
    w, perm = torch.rand(M, generator=g), torch.randperm(M, generator=g).to(torch.int32)
    kept = tuning.Checkpoint8(codes.cuda(), e.cuda())
    gate = None if act == RELU2 else v[0]
    h, hg, hu = act64(act, gate, v[-1], dt)
    th, tg, tu = act_tol(act, gate, v[-1], dt)
    d = dh.double()
    for weights in (True, False):
        got = tuning.activation_backward(kept, dh.cuda(), act, ALPHA, LIMIT, topk_weight=w.cuda() if weights else None,
                                         perm=perm.cuda() if weights else None, want_h=True)
        r = w.to(dt).double()[perm.long()][:, None] if weights else torch.ones(M, 1, dtype=torch.float64)
        close(got.h, h, th, "h")
        close(got.d_up, r * d * hu, (r * d * tu).abs() + (r * d * hu).abs() * 3 * U, "d_up")
        if act == RELU2:
            assert got.d_gate is None
        else:
            close(got.d_gate, r * d * hg, (r * d * tg).abs() + (r * d * hg).abs() * 3 * U, "d_gate")
        if weights:
            dw, tw = torch.zeros(M, dtype=torch.float64), torch.zeros(M, dtype=torch.float64)
            dw[perm.long()] = (d * h).sum(1)
            tw[perm.long()] = (d.abs() * (th + h.abs() * (n + 4) * U)).sum(1)
            close(got.d_weight, dw, tw, "d_weight")
        else:
            assert got.d_weight is None


@pytest.mark.parametrize("dt", [BF16, F32])
def test_activation_limit_slopes(dt):
    """At a limit the slope is the inner one, past it 0."""
    g = torch.tensor([7.0, 7.5, -7.0, -9.0, 6.5, 0.0, 7.0, 1.0] * 4)[None]
    u = torch.tensor([7.0, 1.0, -7.0, 7.5, -7.5, 7.0, -7.0, 0.5] * 4)[None]
    _, kept = tuning.activation_save(g.to(dt).cuda(), u.to(dt).cuda(), GPTOSS, ALPHA, LIMIT)
    v = kept.restore(F32).double().cpu()
    assert torch.equal(v[0], g.double()) and torch.equal(v[1], u.double())
    got = tuning.activation_backward(kept, torch.ones(1, 32, dtype=dt).cuda(), GPTOSS, ALPHA, LIMIT)
    _, hg, hu = act64(GPTOSS, v[0], v[1], dt)
    _, tg, tu = act_tol(GPTOSS, v[0], v[1], dt)
    close(got.d_gate, hg, tg, "d_gate")
    close(got.d_up, hu, tu, "d_up")
    assert (got.d_gate.cpu()[g > 7] == 0).all() and (got.d_up.cpu()[u.abs() > 7] == 0).all()


@pytest.mark.parametrize("act", [SWIGLU, GPTOSS, GEGLU])
def test_activation_far_values(act):
    """Large inputs give the limits of the slopes, not NaN."""
    g = torch.tensor([-1e30, -1e20, -300.0, -90.0, 90.0, 300.0, 1e20, 1e30]).repeat_interleave(32).reshape(8, 32)
    u = torch.full((8, 32), 0.5)
    _, kept = tuning.activation_save(g.cuda(), u.cuda(), act, ALPHA, LIMIT)
    got = tuning.activation_backward(kept, torch.ones(8, 32).cuda(), act, ALPHA, LIMIT, want_h=True)
    for t in (got.d_gate, got.d_up, got.h):
        assert t.isfinite().all()
    top = 0.0 if act == GPTOSS else 0.5
    assert torch.equal(got.d_gate.cpu()[4:], torch.full((4, 32), top)) and (got.d_gate[:4].abs() < 1e-30).all()


@pytest.mark.parametrize("act", [SWIGLU, GPTOSS, GEGLU, RELU2])
def test_activation_rows(act):
    """Rows behind the plan's last stay as they are, a NaN stays in its row, a
    position without a pick has no weight, and dh's place may be taken."""
    M, n, dt = 21, 96, BF16
    v, g = projections(act, M, n, dt, 4), gen(9)
    v[-1, 3, 40] = float("nan")
    parts = len(v)
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    count = torch.tensor([13], dtype=torch.int32).cuda()
    dev = [t.cuda() for t in v]
    out = torch.full((M, n), 7.0, dtype=dt, device="cuda")
    codes = torch.full((parts, M, n), 55, dtype=torch.int8, device="cuda")
    e = torch.full((parts, M, n // 32), 99, dtype=torch.uint8, device="cuda")
    gp = None if act == RELU2 else dev[0].data_ptr()
    check(lib.moe_activation_save(gp, dev[-1].data_ptr(), M, n, moe_dtype(dt), act, ALPHA, LIMIT, count.data_ptr(), out.data_ptr(),
                                  codes.data_ptr(), e.data_ptr(), st))
    whole = tuning.activation_save(None if act == RELU2 else dev[0], dev[-1], act, ALPHA, LIMIT)
    assert same_bits(out[:13], whole[0][:13]) and (out[13:] == 7).all()
    assert torch.equal(codes[:, :13], whole[1].codes[:, :13]) and (codes[:, 13:] == 55).all()
    assert torch.equal(e[:, :13], whole[1].scales[:, :13]) and (e[:, 13:] == 99).all()

    dh = (torch.randn(M, n, generator=g) * 0.01).to(dt).cuda()
    w, perm = torch.rand(M, generator=g).cuda(), torch.randperm(M, generator=g).to(torch.int32)
    clean = tuning.activation_backward(whole[1], dh, act, ALPHA, LIMIT, topk_weight=w, perm=perm.cuda())
    lost = int(perm[5])
    perm[5] = M
    offsets = torch.tensor([0, 4, 13], dtype=torch.int32).cuda()
    got = tuning.activation_backward(whole[1], dh, act, ALPHA, LIMIT, topk_weight=w, perm=perm.cuda(), offsets=offsets)
    for a, b in ((got.d_up, clean.d_up), (got.d_gate, clean.d_gate)):
        if a is None:
            continue
        if a is not got.d_up or act in (RELU2, GPTOSS):  # (a plain product's slope in up does not depend on up)
            assert a[3].isnan().any()
        assert a[[i for i in range(13) if i != 3]].isfinite().all()
        same = [i for i in range(13) if i not in (3, 5)]
        assert same_bits(a[same], b[same]) and (a[5] == 0).all()
    named = [int(p) for i, p in enumerate(perm[:13]) if i not in (3, 5)]
    others = [i for i in range(M) if i not in named and i != int(perm[3])]
    assert same_bits(got.d_weight[named], clean.d_weight[named]) and got.d_weight[int(perm[3])].isnan()
    assert (got.d_weight[others] == 0).all() and lost in others

    # in dh's place
    place = dh.clone()
    other = torch.empty_like(dh)
    dw = torch.empty_like(w)
    perm[5] = lost
    pp = perm.cuda()
    kept = whole[1]
    dg, du = (None, place) if act == RELU2 else (place, other)
    check(lib.moe_activation_backward(kept.codes.data_ptr(), kept.scales.data_ptr(), place.data_ptr(), M, n, moe_dtype(dt), act,
                                      ALPHA, LIMIT, w.data_ptr(), pp.data_ptr(), None, None if dg is None else dg.data_ptr(),
                                      du.data_ptr(), dw.data_ptr(), None, st))
    fine = torch.arange(M, device="cuda") != 3
    assert same_bits(du[fine], clean.d_up[fine]) and (dg is None or same_bits(dg[fine], clean.d_gate[fine]))


# ---------------------------------------------------------- rows and norm --

@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,k,H,add", [(1, 1, 8, False), (1, 8, 2048, True), (3, 2, 24, True), (37, 4, 2880, True), (130, 3, 264, False),
                                       (64, 10, 520, True), (1000, 17, 64, False), (5, 64, 4096, True)])
def test_permute_backward(dt, T, k, H, add):
    g = gen(T * k)
    dX = torch.randn(T * k, H, generator=g).to(dt)
    dx = torch.randn(T, H, generator=g).to(dt) if add else None
    inv = torch.randperm(T * k, generator=g).to(torch.int32).reshape(T, k)
    if T > 4:
        inv = torch.where(torch.rand(T, k, generator=g) < 0.2, torch.full_like(inv, -1), inv)
        inv[2] = -1  # a token that no expert took
        inv[3, 0] = T * k
    on = (inv >= 0) & (inv < T * k)
    rows = torch.where(on[..., None], dX.double()[inv.long().clamp(0, T * k - 1)], 0.0)
    base = dx.double() if add else torch.zeros(T, H, dtype=torch.float64)
    got = tuning.permute_backward(dX.cuda(), inv.cuda(), dx=cuda(dx), out=torch.empty(T, H, dtype=dt).cuda())
    close(got, base + rows.sum(1), (rows.abs().sum(1) + base.abs()) * (k + 1) * U, "dx")
    if add:
        into = dx.cuda()
        assert tuning.permute_backward(dX.cuda(), inv.cuda(), dx=into) is into and same_bits(into, got)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,H,skip", [(1, 8, False), (1, 2048, True), (2, 1024, True), (5, 2880, True), (37, 520, False), (50, 1024, False),
                                      (130, 4096, True), (700, 264, True), (33, 8192, True), (4100, 72, False), (513, 6152, True)])
def test_add_rmsnorm_backward(dt, T, H, skip):
    g = gen(T + H)
    r = (torch.randn(T, H, generator=g) * torch.exp(torch.randn(T, 1, generator=g))).to(dt)
    if T > 2:
        r[1] = 0  # a row of zeros: 1 / sqrt(eps)
    w = (1 + 0.3 * torch.randn(H, generator=g)).to(dt)
    dn = (torch.randn(T, H, generator=g) * 0.01).to(dt)
    dr = (torch.randn(T, H, generator=g) * 0.01).to(dt) if skip else None
    eps = 1e-6
    din, dw = tuning.add_rmsnorm_backward(r.cuda(), w.cuda(), dn.cuda(), eps, d_residual=cuda(dr))
    x, W, d = r.double(), w.double(), dn.double()
    s = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    n, p = x * s, d * W
    m = (p * n).mean(1, keepdim=True)
    base = dr.double() if skip else torch.zeros_like(x)
    c = (H / 2 + 16) * U  # s: half of the mean square's error and a few roundings
    mm = (p * n).abs().mean(1, keepdim=True)
    tol = s * ((p.abs() + n.abs() * mm) * (c + 8 * U) + n.abs() * mm * (H + c) * U + n.abs() * mm * c) + base.abs() * U
    close(din, base + s * (p - n * m), tol, "d_in")
    close(dw, (d * n).sum(0), (d * n).abs().sum(0) * (c + (T + 8) * U), "d_weight")
    # in place of either gradient, and the same bits again
    for at in ("d_normed", "d_residual") if skip else ("d_normed",):
        a, b = dn.cuda(), cuda(dr)
        got, dw2 = tuning.add_rmsnorm_backward(r.cuda(), w.cuda(), a, eps, d_residual=b, out=a if at == "d_normed" else b)
        assert same_bits(got, din) and same_bits(dw2, dw)


def test_add_rmsnorm_backward_of_the_forward():
    """The gradient at the forward's own residual, against differences of the
    forward's definition."""
    T, H, eps = 6, 64, 1e-5
    g = gen(1)
    a, b, w = torch.randn(T, H, generator=g), torch.randn(T, H, generator=g), 1 + 0.2 * torch.randn(H, generator=g)
    ac, bc, wc = a.cuda(), b.cuda(), w.cuda()
    res, xn = torch.empty_like(ac), torch.empty_like(ac)
    check(_lib.load().moe_add_rmsnorm(ac.data_ptr(), bc.data_ptr(), wc.data_ptr(), eps, T, H, _lib.MOE_F32, res.data_ptr(),
                                      xn.data_ptr(), torch.cuda.current_stream().cuda_stream))
    cn, cr = torch.randn(T, H, generator=g), torch.randn(T, H, generator=g)
    din, dw = tuning.add_rmsnorm_backward(res, wc, cn.cuda(), eps, d_residual=cr.cuda())

    def loss(a, w):
        r = a + b.double()
        return (cn.double() * r / torch.sqrt((r * r).mean(1, keepdim=True) + eps) * w).sum() + (cr.double() * r).sum()

    step = 1e-6
    for k in range(12):
        d = torch.randn(T, H, generator=g, dtype=torch.float64)
        slope = (loss(a.double() + step * d, w.double()) - loss(a.double() - step * d, w.double())) / (2 * step)
        assert abs(float((din.double().cpu() * d).sum() - slope)) < 1e-4 * float((din.double().cpu() * d).abs().sum())
        v = torch.randn(H, generator=g, dtype=torch.float64)
        slope = (loss(a.double(), w.double() + step * v) - loss(a.double(), w.double() - step * v)) / (2 * step)
        assert abs(float((dw.double().cpu() * v).sum() - slope)) < 1e-4 * float((dw.double().cpu() * v).abs().sum())


# ------------------------------------------------------------------ chain --

def experts64(x, idx, wt, Wg, Wu, Wd, bd, act, E):
    """The experts' sum for every token in float64, differentiable."""
    y = torch.zeros(x.shape[0], Wd.shape[1], dtype=torch.float64)
    for s in range(idx.shape[1]):
        for e in range(E):
            t = (idx[:, s] == e).nonzero()[:, 0]
            if not len(t):
                continue
            u = x[t] @ Wu[e].t()
            g = None if Wg is None else x[t] @ Wg[e].t()
            o = act64(act, g, u, F32)[0] @ Wd[e].t()
            if bd is not None:
                o = o + bd[e]
            y = y.index_add(0, t, wt[t, s:s + 1] * o)
    return y


def experts(act, E, I, H, bits, gs, dt, bias=False, down_bits=None):
    up, Wu = stack(E, I, H, bits, gs, dt, 1)
    gate, Wg = (None, None) if act == RELU2 else stack(E, I, H, bits, gs, dt, 2)
    down, Wd = stack(E, H, I, down_bits or bits, 32, dt, 3)
    bd = None
    if bias:
        bd = (torch.randn(E, H, generator=gen(4)) * 0.1).to(dt)
        down.out_bias = bd.cuda()
        bd = bd.double()
    return tuning.FrozenExperts(gate, up, down, act, ALPHA, LIMIT), (Wg, Wu, Wd, bd)


@pytest.mark.parametrize("act,bias,kind", [(SWIGLU, False, "even"), (GPTOSS, True, "some"), (GEGLU, False, "one"), (RELU2, False, "some")])
@pytest.mark.parametrize("T", [1, 50])
def test_experts_chain(act, bias, kind, T):
    """A layer's experts forward and backward in f32: within the 8-bit
    checkpoint's effect of the gradient that autograd finds."""
    E, k, I, H = 6, 2, 96, 128
    ex, W = experts(act, E, I, H, 4, 64, F32, bias, 8)
    idx = picks(T, E, k, 3, kind)
    g = gen(2)
    x, wt, d = torch.randn(T, H, generator=g) * 0.5, torch.rand(T, k, generator=g), torch.randn(T, H, generator=g) * 0.1
    base = torch.randn(T, H, generator=g) * 0.1
    y, kept = ex.forward(x.cuda(), idx.cuda(), wt.cuda())
    dx, dw = ex.backward(d.cuda(), kept, dx=base.cuda())
    x64, w64 = x.double().requires_grad_(True), wt.double().requires_grad_(True)
    ref = experts64(x64, idx, w64, *W, act, E)
    assert (y.double().cpu() - ref).abs().max() < 1e-4 * (ref.abs().max() + 1)
    gx, gw = torch.autograd.grad((ref * d.double()).sum(), [x64, w64], allow_unused=True)
    # inputs off by up to 2^-8 of a block's largest move slopes of order 1 by as
    # much: 2 % of the whole gradient is beyond what they can do
    for got, want, what in ((dx.cpu().double() - base.double(), gx, "dx"), (dw.cpu().double(), gw, "dw")):
        off, size = (got - want).norm(), want.norm()
        assert off <= 0.02 * size + 1e-6, f"{what}: {off} of {size}"
    gone = (idx < 0)
    assert (dw.cpu()[gone] == 0).all()


@pytest.mark.parametrize("dt", [BF16, F16])
def test_experts_formats(dt):
    """Gate and up of two formats give what their two gradients give, and the
    chain is what its parts are."""
    E, k, I, H, T = 5, 2, 64, 128, 40
    up, _ = stack(E, I, H, 4, 64, dt, 1)
    gate, _ = stack(E, I, H, 8, 32, dt, 2)
    down, _ = stack(E, H, I, 6, 64, dt, 3)
    ex = tuning.FrozenExperts(gate, up, down)
    idx, g = picks(T, E, k, 3), gen(3)
    x, wt, d = (torch.randn(T, H, generator=g) * 0.5).to(dt).cuda(), torch.rand(T, k, generator=g).cuda(), (torch.randn(T, H, generator=g) * 0.1).to(dt).cuda()
    _, kept = ex.forward(x, idx.cuda(), wt)
    dx, dw = ex.backward(d, kept)
    dh = tuning.expert_matmul_backward(down, d, kept.offsets, perm=kept.perm, top_k=k)
    a = tuning.activation_backward(kept.kept, dh, topk_weight=wt, perm=kept.perm)
    dX = tuning.expert_matmul_backward(gate, a.d_gate, kept.offsets)
    dX = tuning.expert_matmul_backward(up, a.d_up, kept.offsets, dx=dX)
    assert same_bits(dw, a.d_weight) and same_bits(dx, tuning.permute_backward(dX, kept.inv_perm))


def test_experts_captured():
    """Forward and backward in a graph, replayed with new inputs between eager
    calls: every replay gives the eager bits."""
    E, k, I, H, T, dt = 8, 2, 128, 256, 200, BF16
    ex, _ = experts(SWIGLU, E, I, H, 4, 64, dt)
    r, w = torch.randn(T, H).to(dt).cuda(), torch.ones(H, dtype=dt).cuda()

    def step(x, idx, wt, d):
        y, kept = ex.forward(x, idx, wt)
        dx, dw = ex.backward(d, kept)
        din, dn = tuning.add_rmsnorm_backward(r, w, dx, 1e-6, d_residual=d)
        return y, dx, dw, din, dn

    def inputs(seed):
        g = gen(seed)
        return [(torch.randn(T, H, generator=g) * 0.5).to(dt).cuda(), picks(T, E, k, seed, "some").cuda(), torch.rand(T, k, generator=g).cuda(),
                (torch.randn(T, H, generator=g) * 0.1).to(dt).cuda()]

    held = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(*held)
    for seed in range(1, 5):
        new = inputs(seed)
        eager = step(*new)
        for h, t in zip(held, new):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for a, b, what in zip(results, eager, ("y", "dx", "dw", "d_in", "d_weight")):
            assert same_bits(a, b), f"replay {seed}: {what}"


def test_experts_on_a_stream():
    """Calls on a stream of the caller's give the bits of the current one's."""
    ex, _ = experts(SWIGLU, 8, 128, 256, 4, 64, BF16)
    g = gen(1)
    x, idx, wt = torch.randn(90, 256, generator=g).to(BF16).cuda(), picks(90, 8, 2, 1).cuda(), torch.rand(90, 2, generator=g).cuda()
    y, kept = ex.forward(x, idx, wt)
    dx, dw = ex.backward(x, kept)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y2, kept2 = ex.forward(x, idx, wt, stream=side)
    dx2, dw2 = ex.backward(x, kept2, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert same_bits(y, y2) and same_bits(dx, dx2) and same_bits(dw, dw2)


def test_wrappers_refuse():
    x = torch.randn(4, 64, device="cuda")
    p, _ = stack(2, 64, 64, 4, 64, F32, 1)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for kw in (dict(perm=off), dict(proj2=p), dict(dx=x.half()), dict(out=x[:2]), dict(offsets=off.cpu()), dict(offsets=off.long()),
               dict(dy=x[:, :32].contiguous()), dict(dy=x.t().contiguous().t()), dict(dx=x.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            tuning.expert_matmul_backward(**{**dict(proj=p, dy=x, offsets=off), **kw})
    with pytest.raises(MoeError):  # the gradient's own place
        tuning.expert_matmul_backward(p, x, off, out=x)
    with pytest.raises(ValueError):
        tuning.activation_save(None, x, SWIGLU)
    with pytest.raises(ValueError):
        tuning.activation_save(x, x, RELU2)
    with pytest.raises(ValueError):
        tuning.activation_save(x.clone().requires_grad_(True), x)
    with pytest.raises(MoeError):
        tuning.activation_save(x[:, :48].contiguous(), x[:, :48].contiguous())
    h, kept = tuning.activation_save(x, x)
    for bad in (dict(dh=x[:2]), dict(dh=x.cpu()), dict(topk_weight=x[0]), dict(perm=off), dict(kept=tuning.Checkpoint8(kept.codes[:1], kept.scales[:1])),
                dict(offsets=off[:1])):
        with pytest.raises(ValueError):
            tuning.activation_backward(**{**dict(kept=kept, dh=x), **bad})
    with pytest.raises(ValueError):
        kept.restore(torch.float64)
    with pytest.raises(ValueError):
        tuning.permute_backward(x, off)
    with pytest.raises(ValueError):
        tuning.add_rmsnorm_backward(x, x[0, :32], x, 1e-6)
    with pytest.raises(MoeError):
        tuning.add_rmsnorm_backward(x, x[0].clone(), x.clone(), float("nan"))
    with pytest.raises(ValueError):
        tuning.FrozenExperts(p, p, stack(2, 32, 64, 4, 64, F32, 1)[0])
