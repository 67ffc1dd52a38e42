"""What the gradients through the experts keep of their inputs: weights, sums and slopes to fp32's precision,
kept values in every type, rows apart from one another."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_expert_grad import (ALPHA, CASES, GPTOSS, LIMIT, RELU2, SWIGLU, act64, act_tol, grad64, half, picks,  # noqa: E402
                                  plan, stack)
from test_gpu_tuning import BF16, F16, F32, U, close, cuda, gen, same_bits  # noqa: E402

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd.layer import StackedExperts  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    _lib.load()
    yield
    torch.cuda.synchronize()


def packed(q, s, b, bits, gs):
    """A stack of codes q [E, N, K] with scales and biases [E, N, K / gs]."""
    E, N, K = q.shape
    stream = ((q[..., None] >> torch.arange(bits)) & 1).reshape(E, N, K * bits // 32, 32)
    w = (stream.long() << torch.arange(32)).sum(-1)
    return StackedExperts(torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32).cuda(), s.cuda(), b.cuda(), bits, gs)


# rows that take the kernels of few rows (narrow blocks twice, wide ones), of 128 and of 256 rows
ROWS = [(8, 30), (64, 100), (64, 1500), (4, 900), (40, 2000)]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("bits", [2, 3, 4, 5, 6, 8])
@pytest.mark.parametrize("E,T", ROWS)
def test_weights_that_differ_in_their_last_bits(dt, bits, E, T):
    """Weights 1 + q 2^-10 (bf16) or 1 + q 2^-13 (f16), whose bits pass the type's: the difference of two, which the
    type holds, comes out exactly."""
    N, K, gs = 104, 2080, 32
    low = -10 if dt == BF16 else -13
    g = gen(bits)
    q = torch.randint(0, 2 ** bits, (E, N, K), generator=g)
    s, b = torch.full((E, N, K // gs), 2.0 ** low, dtype=dt), torch.ones(E, N, K // gs, dtype=dt)
    p = packed(q, s, b, bits, gs)
    _, _, offsets = plan(picks(T, E, 1, 5), E)
    at = torch.stack([torch.randperm(N, generator=g)[:2] for _ in range(T)])
    dy = torch.zeros(T, N).scatter_(1, at[:, :1], 1.0).scatter_(1, at[:, 1:], -1.0).to(dt)
    e = torch.searchsorted(offsets[1:].long(), torch.arange(T), right=True)
    ref = (q[e, at[:, 0]] - q[e, at[:, 1]]).double() * 2.0 ** low
    for kw in ({}, dict(proj2=p, dy2=dy.cuda())):
        got = tuning.expert_matmul_backward(p, dy.cuda(), offsets.cuda(), **kw)
        assert torch.equal(got.cpu().double(), ref * (2 if kw else 1))


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("T,E,k,N,K,bits,gs,pair,gather,add,kind", CASES)
def test_products_keep_their_weights(dt, T, E, k, N, K, bits, gs, pair, gather, add, kind):
    """A weight enters as two values of the type: the second is off by at most half a step of at most half a step, 2^-16
    (bf16) or 2^-22 (f16, there 2^-25 at least) of the weight. Sums are fp32."""
    M, g = T * k, gen(T + N)
    sb = dt if T != 37 else (F16 if dt == BF16 else BF16)
    stacks = [stack(E, N, K, bits, gs, sb, 7 * i + E) for i in range(2 if pair else 1)]
    perm, _, offsets = plan(picks(T, E, k, T, kind), E)
    if not gather:
        perm = None
    dys = [(torch.randn(T if gather else M, N, generator=g) * 0.01).to(dt) for _ in stacks]
    base = (torch.randn(M, K, generator=g) * 0.01).to(dt) if add else torch.zeros(M, K, dtype=dt)
    ref, mag, only = grad64([w for _, w in stacks], dys, offsets, perm, k, base)
    kw = dict(perm=cuda(perm), top_k=k, dx=base.cuda() if add else None, out=torch.zeros(M, K, dtype=dt).cuda())
    if pair:
        kw.update(proj2=stacks[1][0], dy2=dys[1].cuda())
    got = tuning.expert_matmul_backward(stacks[0][0], dys[0].cuda(), offsets.cuda(), **kw)
    used, n = int(offsets[-1]), N * len(stacks)
    two = torch.finfo(dt).eps ** 2 / 4
    tol = mag * (two + (2 * n + 8) * U) + only * (2.0 ** -25 if dt == F16 else 0.0) + base.double().abs() * 2 * U
    close(got[:used], ref[:used], tol[:used], "dx")


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("E,T", ROWS)
def test_infinities_come_out_as_such(dt, E, T):
    """An infinite gradient or weight gives infinities of its sign, as the sum has them, not NaN."""
    N, K, gs = 64, 2080, 32
    q = torch.randint(1, 16, (E, N, K), generator=gen(1))
    s, b = torch.full((E, N, K // gs), 2.0 ** -10, dtype=dt), torch.full((E, N, K // gs), 0.75, dtype=dt)
    p = packed(q, s, b, 4, gs)
    _, _, offsets = plan(picks(T, E, 1, 5), E)
    dy = torch.ones(T, N, dtype=dt)
    plain = tuning.expert_matmul_backward(p, dy.cuda(), offsets.cuda())
    dy[0, 3], dy[T - 1, 50] = float("inf"), float("-inf")
    got = tuning.expert_matmul_backward(p, dy.cuda(), offsets.cuda())
    assert (got[0] == float("inf")).all() and (got[T - 1] == float("-inf")).all()
    assert same_bits(got[1:T - 1], plain[1:T - 1])
    last = int((offsets[1:] > offsets[:-1]).nonzero().max())
    p.biases[last, 9, 1] = float("-inf")
    got = tuning.expert_matmul_backward(p, torch.ones(T, N, dtype=dt).cuda(), offsets.cuda())
    a = int(offsets[last])
    assert (got[a:, 32:64] == float("-inf")).all() and same_bits(got[:a], plain[:a])
    assert same_bits(got[a:, :32], plain[a:, :32]) and same_bits(got[a:, 64:], plain[a:, 64:])


def test_wide_rows_of_many_experts():
    """Just past the few-row kernel's rows, 1024 experts of 2^20 columns: more column blocks than one launch holds."""
    if torch.cuda.mem_get_info()[0] < 130 << 30:
        pytest.skip("needs 130 GB")
    E, N, K, M = 1024, 8, 1 << 20, 45100
    w = torch.randint(-2 ** 31, 2 ** 31 - 1, (1, N, K // 16), dtype=torch.int64, generator=gen(1)).to(torch.int32)
    w = w.cuda().repeat(E, 1, 1)
    s = torch.full((E, N, K // 128), 2.0 ** -6, dtype=BF16, device="cuda")
    b = torch.arange(E, device="cuda").to(BF16)[:, None, None].expand(E, N, K // 128).contiguous()
    p = StackedExperts(w, s, b, 2, 128)
    offsets = torch.linspace(0, M, E + 1, dtype=torch.float64).round().to(torch.int32)
    dy = (torch.arange(M * N) % 7 - 3).reshape(M, N).to(BF16)
    dx = tuning.expert_matmul_backward(p, dy.cuda(), offsets.cuda())
    q = (w[0, :, :, None] >> (2 * torch.arange(16, device="cuda"))) & 3
    q = q.reshape(N, K).double()
    for row in (0, 44, 22550, M - 1):
        e = int(torch.searchsorted(offsets[1:].long(), torch.tensor(row), right=True))
        d = dy[row].double().cuda()
        ref = d @ (q * 2.0 ** -6 + b[e, 0, 0].double())
        mag = d.abs() @ (q * 2.0 ** -6 + b[e, 0, 0].double())
        close(dx[row], ref, mag.cpu() * (2.0 ** -16 + 32 * U), f"row {row}")
    del dx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("bits", [3, 4, 8])
@pytest.mark.parametrize("E,T", ROWS)
def test_infinities_added_in_place(dt, bits, E, T):
    """What is not finite is added to dx once, and what is finite beside it keeps its bits: in dx's own place, apart from
    it, and in a replayed graph."""
    N, K = 72, 2080
    p, _ = stack(E, N, K, bits, 32, dt, 3)
    _, _, offsets = plan(picks(T, E, 1, 5), E)
    g = gen(1)
    dy, base = (torch.randn(T, N, generator=g) * 0.01).to(dt).cuda(), (torch.randn(T, K, generator=g) * 0.01).to(dt).cuda()
    off = offsets.cuda()
    plain = tuning.expert_matmul_backward(p, dy, off, dx=base, out=torch.empty_like(base))
    bad = dy.clone()
    bad[T // 2, 70], bad[T - 1, 3] = float("inf"), float("nan")
    last = int((offsets[1:] > offsets[:-1]).nonzero().max())
    p.scales[last, 9, 2] = float("inf")
    apart = tuning.expert_matmul_backward(p, bad, off, dx=base, out=torch.empty_like(base))
    place = base.clone()
    assert same_bits(tuning.expert_matmul_backward(p, bad, off, dx=place), apart)
    ok = torch.ones(T, K, dtype=torch.bool)
    ok[[T // 2, T - 1]] = False
    ok[int(offsets[last]):, 64:96] = False
    ok = ok.cuda()
    assert same_bits(apart[ok], plain[ok]) and not apart[~ok].isfinite().any()
    held = bad.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tuning.expert_matmul_backward(p, held, off, dx=base, out=place)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tuning.expert_matmul_backward(p, held, off, dx=base, out=place)
    clean = tuning.expert_matmul_backward(p, dy, off, dx=base, out=torch.empty_like(base))
    for rows, want in ((bad, apart), (dy, clean), (bad, apart)):
        held.copy_(rows)
        place.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert same_bits(place, want)


@pytest.mark.parametrize("E,T", ROWS)
def test_weights_past_f16(E, T):
    """bf16 scales beside f16 rows: a weight of 65504 is itself, one of 65520 or more infinite, in every kernel."""
    N, K = 64, 2080
    s, b = torch.zeros(E, N, K // 32, dtype=BF16), torch.ones(E, N, K // 32, dtype=BF16)
    s[:, :, 1], b[:, :, 1] = 16.0, 65280.0  # 65280, 65296, ... 65504, 65520
    b[:, :, 2] = 70144.0
    q = (torch.arange(K) % 16).expand(E, N, K).contiguous()
    p = packed(q, s, b, 4, 32)
    _, _, offsets = plan(picks(T, E, 1, 5), E)
    dy = torch.zeros(T, N, dtype=F16)
    dy[:, 7] = 0.5
    w = 65280.0 + 16.0 * q[0, 0, 32:64].double()
    # (beside 0.5 the rows are 0, and 0 times an infinite weight is NaN; of 64 values of 2^-7 the sum is w / 2 too)
    for rows, past in ((dy, float("nan")), (torch.full((T, N), 2.0 ** -7, dtype=F16), float("inf"))):
        got = tuning.expert_matmul_backward(p, rows.cuda(), offsets.cuda())
        ref = torch.full((K,), 0.5, dtype=torch.float64)
        ref[32:64], ref[64:96] = torch.where(w < 65520, w / 2, past), past
        close(got, ref.expand(T, K), 0.0, "dx")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("N", [8, 56, 72, 104])
@pytest.mark.parametrize("E,T", ROWS)
def test_infinity_in_the_last_values_of_a_row(dt, N, E, T):
    """Of n values that end inside a chunk: weights of one sign give the infinity, whatever the number of rows."""
    K = 2080
    q = torch.randint(0, 16, (E, N, K), generator=gen(N))
    p = packed(q, torch.full((E, N, K // 32), 2.0 ** -6, dtype=dt), torch.ones(E, N, K // 32, dtype=dt), 4, 32)
    _, _, offsets = plan(picks(T, E, 1, 5), E)
    dy = torch.ones(T, N, dtype=dt)
    plain = tuning.expert_matmul_backward(p, dy.cuda(), offsets.cuda(), proj2=p, dy2=dy.cuda())
    bad, bad2 = dy.clone(), dy.clone()
    bad[T // 2, N - 1], bad2[T - 1, N - 8:] = float("inf"), float("-inf")
    got = tuning.expert_matmul_backward(p, bad.cuda(), offsets.cuda(), proj2=p, dy2=bad2.cuda())
    assert (got[T // 2] == float("inf")).all() and (got[T - 1] == float("-inf")).all()
    keep = torch.ones(T, dtype=torch.bool)
    keep[[T // 2, T - 1]] = False
    assert same_bits(got[keep.cuda()], plain[keep.cuda()])


# ---------------------------------------------------------------- kept values --

@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_the_largest_values_come_back(dt):
    """Finite values of the type's last steps are restored within half a step of their block's: f16 has no 65536."""
    top = {F16: [65504.0, 65472.0, 65280.0, 65248.0, 65024.0, 64992.0, 64512.0],
           BF16: [3.36e38, 3.2e38, 1.7e38], F32: [3.38e38, 3.2e38, 1.7e38]}[dt]
    v = torch.randn(2 * len(top), 32, generator=gen(2)) * (top[0] / 8)
    for i, x in enumerate(top):
        v[2 * i, 5], v[2 * i + 1, 9] = x, -x
    v = v.to(dt)
    _, kept = tuning.activation_save(None, v.cuda(), _lib.MOE_ACT_RELU2)
    back = kept.restore(dt).cpu()[0]
    step = torch.exp2(kept.scales[0].double().cpu() - 133).repeat_interleave(32, -1)
    assert back.isfinite().all() and ((back.double() - v.double()).abs() <= step / 2).all()
    if dt == F16:  # what no f16 row holds is rounded as ever
        far = torch.tensor([[70000.0] + [0.0] * 31])
        _, kept = tuning.activation_save(None, far.cuda(), _lib.MOE_ACT_RELU2)
        assert kept.restore(F16)[0, 0, 0] == float("inf")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_how_far_a_kept_value_is_off(dt):
    """By half a step, and a block's largest is 63.75 steps at least: 2^-6.99 of it. A largest value just above that
    and a tie come to 2^-7, more than 2^-7.98. Where the exponent ends, half of 2^-133."""
    most = 0.5 / 63.75
    g = gen(7)
    top = 1.0 + torch.rand(512, 1, generator=g) ** 4
    v = (torch.rand(512, 32, generator=g) * 2 - 1) * top
    v[:, :1] = top
    v[0], v[1] = 0.0, 0.0
    v[0, 0], v[0, 1] = 1.0, 0.5 + 2.0 ** -7  # 32.5 steps of 2^-6
    v[1, 0], v[1, 1] = 63.75 / 64, 33.5 / 64  # the least that takes this step (in f32, f16)
    v = (v * torch.exp2(torch.randint(-10, 10, (512, 1), generator=g).float())).to(dt)
    _, kept = tuning.activation_save(None, v.cuda(), _lib.MOE_ACT_RELU2)
    off = (kept.restore(F32)[0].double().cpu() - v.double()).abs().amax(1) / v.double().abs().amax(1)
    assert (off <= most).all() and off[0] == 2.0 ** -7
    if dt != F16:  # f16 has no value so small
        v = torch.zeros(3, 32)
        v[0, 0], v[1, 0], v[1, 1], v[2, 0], v[2, 1] = 2.0 ** -133, 2.0 ** -127, 2.0 ** -133, 1.5 * 2.0 ** -132, 1.5 * 2.0 ** -133
        v = v.to(dt)
        _, kept = tuning.activation_save(None, v.cuda(), _lib.MOE_ACT_RELU2)
        assert (kept.scales == 0).all()
        assert ((kept.restore(F32)[0].double().cpu() - v.double()).abs() <= 2.0 ** -134).all()


# ------------------------------------------------------------- the weights' gradient --

def test_a_pick_that_no_row_names_has_no_gradient():
    """A perm entry past M, with and without the plan's offsets: the pick it does not name gets zero, not what lay in
    the memory."""
    M, n = 4096, 64
    _, kept = tuning.activation_save(torch.randn(M, n, device="cuda"), torch.randn(M, n, device="cuda"))
    dh, w = torch.randn(M, n, device="cuda"), torch.rand(M, device="cuda")
    perm = torch.randperm(M, generator=gen(1)).to(torch.int32)
    lost = [int(perm[5]), int(perm[4000])]
    perm[5], perm[4000] = M, -1
    rest = torch.ones(M, dtype=torch.bool)
    rest[lost] = False
    for offsets in (None, torch.tensor([0, 7, M], dtype=torch.int32).cuda()):
        for _ in range(4):
            dirt = [torch.full((M,), float("nan"), device="cuda") for _ in range(8)]
            del dirt
            dw = tuning.activation_backward(kept, dh, topk_weight=w, perm=perm.cuda(), offsets=offsets).d_weight.cpu()
            assert (dw[lost] == 0).all() and (dw[rest] != 0).any() and dw.isfinite().all()


# ------------------------------------------------------------------------- sums --

@pytest.mark.parametrize("T", [3, 130])
def test_long_sums_in_f32(T):
    """8192 values of 1 + 2^-15, twice: a sum that takes them one after another loses their last bits from 2^11 on."""
    N, K = 8192, 64
    p = packed(torch.zeros(1, N, K, dtype=torch.int64), torch.ones(1, N, 2), torch.full((1, N, 2), 1 + 2.0 ** -15), 4, 32)
    dy, offsets = torch.ones(T, N, device="cuda"), torch.tensor([0, T], dtype=torch.int32, device="cuda")
    assert (tuning.expert_matmul_backward(p, dy, offsets) == 8192.25).all()
    assert (tuning.expert_matmul_backward(p, dy, offsets, proj2=p, dy2=dy) == 16384.5).all()


@pytest.mark.parametrize("pair", [False, True])
def test_sums_in_f32_stay_short(pair):
    """A chunk's 32 values, the chunks one after another and a few roundings more, of the sum of magnitudes."""
    T, E, N, K = 90, 3, 4100 - 4, 96
    stacks = [stack(E, N, K, 6, 32, F32, i) for i in range(1 + pair)]
    _, _, offsets = plan(picks(T, E, 1, 4), E)
    dys = [torch.rand(T, N, generator=gen(i)) for i in range(1 + pair)]
    zero = torch.zeros(T, K)
    ref, mag, _ = grad64([w for _, w in stacks], dys, offsets, None, 1, zero)
    kw = dict(proj2=stacks[1][0], dy2=dys[1].cuda()) if pair else {}
    got = tuning.expert_matmul_backward(stacks[0][0], dys[0].cuda(), offsets.cuda(), **kw)
    close(got, ref, mag * (32 + len(stacks) * N / 32 + 8) * U, "dx")


# ----------------------------------------------------------------------- slopes --

@pytest.mark.parametrize("act", [_lib.MOE_ACT_SWIGLU, _lib.MOE_ACT_GPTOSS])
def test_slopes_far_from_zero(act):
    """In f32 the logistic of g is off by a dozen roundings wherever it is (an exponential of 2, its two factors, a sum,
    a reciprocal of 2, three products), and by |alpha g| of them for the rounded product alpha g that it is taken of;
    not by |g| again for the exponential's own."""
    g = torch.linspace(-84, 84, 32 * 256).reshape(256, 32)
    if act == _lib.MOE_ACT_GPTOSS:
        g = g / 1.75
    u = torch.rand(256, 32, generator=gen(3)) + 0.5
    _, kept = tuning.activation_save(g.cuda(), u.cuda(), act, 1.702, 1e4)
    v = kept.restore(F32).double().cpu()
    dh = (torch.rand(256, 32, generator=gen(4)) + 0.5)
    got = tuning.activation_backward(kept, dh.cuda(), act, 1.702, 1e4, want_h=True)
    alpha = float(torch.tensor(1.702)) if act == _lib.MOE_ACT_GPTOSS else 1.0
    one = 1.0 if act == _lib.MOE_ACT_GPTOSS else 0.0
    s = torch.sigmoid(alpha * v[0])
    a, c = v[0] * s, (16 + (alpha * v[0].abs() if one else 0.0)) * U
    d, up = dh.double(), v[1] + one
    close(got.d_up, d * a, (d * a).abs() * c, "d_up")
    close(got.h, a * up, (a * up).abs() * c, "h")
    # 1 - s is off by what s is, s (1 - s) by both
    rest = alpha * a * (1 - s)
    size = s + (alpha * a).abs() * ((1 - s) + s)
    close(got.d_gate, d * (s + rest) * up, (d * up).abs() * size * (c + 4 * U), "d_gate")


# ------------------------------------------------------------------------ chain --

@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("act,two_formats,bias", [(SWIGLU, False, False), (SWIGLU, True, False), (GPTOSS, False, True), (RELU2, False, False)])
@pytest.mark.parametrize("T", [1, 61, 700])
def test_experts_in_16_bits(dt, act, two_formats, bias, T):
    """Forward and backward of the chain against float64: the backward at the values kept, every rounding on the way
    counted once."""
    E, k, I, H = 6, 2, 104 - 8, 192
    up, Wu = stack(E, I, H, 4, 64, dt, 1)
    gate, Wg = (None, None) if act == RELU2 else stack(E, I, H, 8 if two_formats else 4, 32 if two_formats else 64, dt, 2)
    down, Wd = stack(E, H, I, 6, 32, dt, 3)
    bd = torch.zeros(E, H, dtype=dt)
    if bias:
        bd = (torch.randn(E, H, generator=gen(4)) * 0.1).to(dt)
        down.out_bias = bd.cuda()
    ex = tuning.FrozenExperts(gate, up, down, act, ALPHA, LIMIT)
    idx, g = picks(T, E, k, 3, "some"), gen(5)
    perm, inv, offsets = plan(idx, E)
    x, wt, d = (torch.randn(T, H, generator=g) * 0.5).to(dt), torch.rand(T, k, generator=g), (torch.randn(T, H, generator=g) * 0.1).to(dt)
    base = (torch.randn(T, H, generator=g) * 0.1).to(dt)
    y, kept = ex.forward(x.cuda(), idx.cuda(), wt.cuda())
    dx, dw = ex.backward(d.cuda(), kept, dx=base.cuda())
    used, hf, two = int(offsets[-1]), half(dt), torch.finfo(dt).eps ** 2 / 4 + (2 * H + 8) * U
    p = perm[:used].long()
    row, e = p // k, torch.searchsorted(offsets[1:].long(), torch.arange(used), right=True)
    tiny = 2.0 ** -25 if dt == F16 else 0.0

    def times(rows, W):  # rows [used, n] by their experts' [n, m]
        out = torch.zeros(used, W.shape[2], dtype=torch.float64)
        for i in range(E):
            out[e == i] = rows[e == i] @ W[i]
        return out

    # forward: the activation's inputs off by a rounding of theirs, of the weights (f16) and half a step more of the
    # value, the experts' rows and their sum a rounding each: 8 half steps of the whole
    xd = x.double()[row]
    gd, ud = None if Wg is None else times(xd, Wg.transpose(1, 2)), times(xd, Wu.transpose(1, 2))
    Y = times(act64(act, gd, ud, F32)[0], Wd.transpose(1, 2)) + bd.double()[e]
    ref = torch.zeros(T, H, dtype=torch.float64).index_add(0, row, wt.double().flatten()[p][:, None] * Y)
    assert (y.double().cpu() - ref).norm() <= 8 * hf * ref.norm()
    # backward
    v = kept.kept.restore(F32).double().cpu()[:, :used]
    gk, uk = None if act == RELU2 else v[0], v[-1]
    h, hg, hu = act64(act, gk, uk, F32)
    th, tg, tu = act_tol(act, gk, uk, F32)
    r = wt.to(dt).double().flatten()[p][:, None]
    D = d.double()[row]
    dh = times(D, Wd)
    off = dh.abs() * hf + times(D.abs(), Wd.abs()) * two + D.abs().sum(1, keepdim=True) * tiny + tiny
    dX, oX = torch.zeros(used, H, dtype=torch.float64), torch.zeros(used, H, dtype=torch.float64)
    for W, slope, ts in ((Wg, hg, tg), (Wu, hu, tu)):
        if W is None:
            continue
        a = r * dh * slope
        oa = (r * slope).abs() * off + (r * dh).abs() * ts + a.abs() * 3 * U
        oa = oa + (a.abs() + oa) * hf + tiny
        dX += times(a, W)
        oX += times(oa, W.abs()) + times(a.abs(), W.abs()) * two + a.abs().sum(1, keepdim=True) * tiny
        if W is Wg and two_formats:  # rounded before the second projection's is added
            oX += (dX.abs() + oX) * hf + tiny
    oX += (dX.abs() + oX) * hf + tiny
    rx, ox = base.double().index_add(0, row, dX), (base.double().abs() * 4 * U).index_add(0, row, oX + dX.abs() * 4 * U)
    close(dx, rx, ox, "dx")
    rw, ow = torch.zeros(T * k, dtype=torch.float64), torch.zeros(T * k, dtype=torch.float64)
    if bias:  # from the experts' rows, which the forward rounded
        Yk = kept.Y[:used].double().cpu()
        rw[p], ow[p] = (D * Yk).sum(1), (D * Yk).abs().sum(1) * (H + 8) * U
    else:
        rw[p], ow[p] = (dh * h).sum(1), (off * h.abs() + dh.abs() * th + (dh * h).abs() * (I + 8) * U).sum(1)
    close(dw.flatten(), rw, ow, "d_weight")
