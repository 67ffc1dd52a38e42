"""Gradients through the experts against differences and adjoints of the forward, and the calls that take another's
place: values written over their inputs, no row at all, a position named twice, two streams at once."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_expert_grad import (ALPHA, GEGLU, GPTOSS, LIMIT, RELU2, SWIGLU, experts, half, picks, plan,  # noqa: E402
                                  stack)
from test_gpu_tuning import BF16, F16, F32, U, cuda, gen, same_bits  # noqa: E402

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd._lib import check  # noqa: E402
from ffai_amd.layer import moe_dtype  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    _lib.load()
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T,E,k,N,K,bits", [(3, 4, 2, 64, 96, 4), (300, 5, 2, 136, 288, 3), (2100, 4, 1, 72, 544, 6)])
def test_product_is_the_forwards_adjoint(dt, T, E, k, N, K, bits):
    """<dy, W x> = <W^T dy, x> for the rows that the forward makes."""
    p, W = stack(E, N, K, bits, 32, dt, T)
    perm, _, offsets = plan(picks(T, E, k, 2), E)
    M, g = T * k, gen(8)
    x, dy = torch.randn(T, K, generator=g).to(dt).cuda(), torch.randn(M, N, generator=g).to(dt).cuda()
    lib, st, off, pm = _lib.load(), torch.cuda.current_stream().cuda_stream, offsets.cuda(), perm.cuda()
    import ctypes as C
    desc = C.byref(p.struct())
    y = torch.empty(M, N, dtype=dt, device="cuda")
    need = lib.moe_expert_matmul_workspace_bytes(desc, moe_dtype(dt), M)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    check(lib.moe_expert_matmul(desc, x.data_ptr(), moe_dtype(dt), pm.data_ptr(), k, M, off.data_ptr(), y.data_ptr(), ws.data_ptr(),
                                need, st))
    dX = tuning.expert_matmul_backward(p, dy, off)
    X = x[pm.long() // k].double()
    here = (dy.double() * y.double()).sum(1)
    there = (dX.double() * X).sum(1)
    mag = torch.empty(M, dtype=torch.float64, device="cuda")
    for e in range(E):
        a, b = int(offsets[e]), int(offsets[e + 1])
        mag[a:b] = (dy[a:b].double().abs() @ W[e].cuda().abs() * X[a:b].abs()).sum(1)
    # each side rounds its weights and its results once (f16 rows in bf16's place: once more), and adds N or K products
    each = 3 * half(dt) if dt != F32 else 3 * U
    assert ((here - there).abs() <= mag * (2 * each + (N + K + 64) * U) + 1e-30).all()


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("E,M,K", [(40, 90, 2048), (4, 700, 544), (70, 9000, 1024)])
def test_a_plan_past_the_rows(dt, E, M, K):
    """Offsets past M end there, and perm's entries past M take the last row: nothing is written behind dx."""
    p, W = stack(E, 64, K, 4, 32, dt, 2)
    dy = torch.randn(M, 64, generator=gen(2)).to(dt).cuda()
    good = torch.linspace(0, M, E + 1).round().to(torch.int32)
    good[-2] = M
    bad = good.clone()
    bad[-2:] = torch.tensor([M + 300, 2 ** 31 - 1])
    perm = torch.randperm(M, generator=gen(3)).to(torch.int32)
    perm[5] = M - 1
    wild = perm.clone()
    wild[5] = -1
    whole = torch.full((M + 600, K), 7.25, dtype=dt, device="cuda")
    a = tuning.expert_matmul_backward(p, dy, good.cuda(), perm=perm.cuda())
    b = tuning.expert_matmul_backward(p, dy, bad.cuda(), perm=wild.cuda(), out=whole[:M])
    assert same_bits(a, b) and (whole[M:] == 7.25).all()


def value(act, g, u):
    """The activation in float64."""
    if act == RELU2:
        return u.clamp(min=0) ** 2
    if act == GPTOSS:
        return g * torch.sigmoid(ALPHA * g) * (u + 1)
    if act == GEGLU:
        return 0.5 * g * (1 + torch.tanh(0.7978845608 * (g + 0.044715 * g ** 3))) * u
    return g * torch.sigmoid(g) * u


@pytest.mark.parametrize("act", [SWIGLU, GPTOSS, GEGLU, RELU2])
def test_activation_matches_differences(act):
    """At the kept values, in f32; below the limit, and squared ReLU away from its bend."""
    M, n, step, g = 33, 160, 2.0 ** -17, gen(5)
    gate, up = ((torch.randn(M, n, generator=g) * 1.2).clamp(-6, 6).cuda() for _ in range(2))
    _, kept = tuning.activation_save(None if act == RELU2 else gate, up, act, ALPHA, LIMIT)
    v = kept.restore(F32).double()
    G, Up = (v[0], v[-1])
    dh = torch.randn(M, n, generator=g).cuda()
    got = tuning.activation_backward(kept, dh, act, ALPHA, LIMIT)
    size = (1 + G.abs()) * (1 + Up.abs())
    # third derivatives are below 8 times size here (step^2 / 6 of them), values below size squared (2^-53 / step of
    # them); the kernel's own slope is off by some tens of roundings of size
    tol = dh.double().abs() * size * (8 * step * step / 6 + 2.0 ** -50 / step * size + 128 * U)
    slope = (value(act, G, Up + step) - value(act, G, Up - step)) / (2 * step)
    smooth = Up.abs() > 2 * step if act == RELU2 else torch.ones_like(Up, dtype=torch.bool)
    assert ((got.d_up.double() - dh.double() * slope).abs() <= tol)[smooth].all()
    if act != RELU2:
        slope = (value(act, G + step, Up) - value(act, G - step, Up)) / (2 * step)
        assert ((got.d_gate.double() - dh.double() * slope).abs() <= tol).all()


@pytest.mark.parametrize("T,H", [(5, 64), (70, 1000), (9, 5000), (70, 2504), (3000, 2176)])
def test_norm_matches_differences(T, H):
    """Along a direction per row and per column, in f32."""
    g, step, eps = gen(H), 2.0 ** -15, 1e-6
    r, d, dr = (torch.randn(T, H, generator=g).cuda() for _ in range(3))
    w = (1 + 0.1 * torch.randn(H, generator=g)).cuda()
    din, dw = tuning.add_rmsnorm_backward(r, w, d, eps, d_residual=dr)
    R, D, DR, Wt = r.double(), d.double(), dr.double(), w.double()

    def terms(R, Wt):
        n = R / torch.sqrt((R * R).mean(1, keepdim=True) + eps)
        return D * n * Wt + DR * R

    along = torch.randn(T, H, generator=g).cuda().double()
    slope = ((terms(R + step * along, Wt) - terms(R - step * along, Wt)) / (2 * step)).sum(1)
    # per element: a slope's sum of magnitudes is that of its terms over r, of order |d w| + |dr|; step^2 / 6 of a
    # third derivative of that order (times the direction's cube), H roundings of the sums
    size = ((D * Wt).abs() * (1 + (D * Wt * R).abs().mean(1, keepdim=True)) * (1 + R.abs()) + DR.abs()) * (1 + along.abs()) ** 3
    tol = size.sum(1) * (10 * step * step + 2.0 ** -50 / step + (H + 64) * U)
    assert ((din.double() * along).sum(1) - slope).abs().le(tol).all()
    turn = torch.randn(H, generator=g).cuda().double()
    slope = ((terms(R, Wt + step * turn) - terms(R, Wt - step * turn)) / (2 * step)).sum(0)
    tol = ((D * R).abs().sum(0) * turn.abs() + (D * R * Wt).abs().sum(0) + (DR * R).abs().sum(0)) * (2.0 ** -50 / step + (H + T + 64) * U)
    assert (dw.double() * turn - slope).abs().le(tol).all()


@pytest.mark.parametrize("act", [SWIGLU, GPTOSS, GEGLU, RELU2])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_save_over_its_inputs(act, dt):
    g = gen(3)
    gate, up = (torch.randn(517, 160, generator=g).to(dt).cuda() for _ in range(2))
    first = None if act == RELU2 else gate
    h, kept = tuning.activation_save(first, up, act, ALPHA, LIMIT)
    for name in ("gate", "up") if act != RELU2 else ("up",):
        a, b = None if first is None else gate.clone(), up.clone()
        place = a if name == "gate" else b
        got, k2 = tuning.activation_save(a, b, act, ALPHA, LIMIT, out=place)
        assert got is place and same_bits(got, h) and torch.equal(k2.codes, kept.codes) and torch.equal(k2.scales, kept.scales)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("E,T", [(64, 100), (4, 900), (40, 2000)])
def test_infinity_at_an_odd_rows_end(dt, E, T):
    """n = 104 ends inside a chunk: an infinity in a row's last values leaves the other rows as they are."""
    N, K = 104, 2080
    p, _ = stack(E, N, K, 4, 32, dt, 3)
    _, _, offsets = plan(picks(T, E, 1, 5), E)
    off = offsets.cuda()
    dy = (torch.randn(T, N, generator=gen(1)) * 0.01).to(dt).cuda()
    plain = tuning.expert_matmul_backward(p, dy, off)
    rows = [0, T // 2, T - 1]
    dy[rows, N - 1] = float("inf")
    got = tuning.expert_matmul_backward(p, dy, off)
    keep = torch.ones(T, dtype=torch.bool)
    keep[rows] = False
    keep = keep.cuda()
    assert same_bits(got[keep], plain[keep]) and not got[~keep].isfinite().any()


@pytest.mark.parametrize("act,bias", [(SWIGLU, False), (GPTOSS, True)])
def test_experts_without_a_pick(act, bias):
    """Picks of no expert alone: nothing comes out and nothing comes back."""
    ex, _ = experts(act, 6, 96, 128, 4, 64, BF16, bias)
    g = gen(1)
    x, wt = torch.randn(40, 128, generator=g).to(BF16).cuda(), torch.rand(40, 2, generator=g).cuda()
    y, kept = ex.forward(x, torch.full((40, 2), -1, dtype=torch.int32).cuda(), wt)
    base = torch.randn(40, 128, generator=g).to(BF16).cuda()
    dx, dw = ex.backward(x, kept, dx=base.clone())
    assert (y == 0).all() and same_bits(dx, base) and (dw == 0).all()


def test_permute_names_a_position_twice():
    """Each naming adds the row: the sum of what is named, in its order."""
    dX = torch.randn(6, 40, generator=gen(1)).cuda()
    inv = torch.tensor([[1, 1], [5, -1], [-1, -1]], dtype=torch.int32).cuda()
    dx = tuning.permute_backward(dX, inv)
    assert torch.equal(dx, torch.stack([dX[1] + dX[1], dX[5], torch.zeros_like(dX[0])]))


def test_two_streams_at_once():
    """Steps of two batches on two streams, several deep, give the bits of one after the other."""
    ex, _ = experts(SWIGLU, 32, 256, 512, 4, 64, BF16)
    r, w = torch.randn(700, 512, generator=gen(9)).to(BF16).cuda(), torch.ones(512, dtype=BF16).cuda()

    def inputs(seed):
        g = gen(seed)
        return [torch.randn(700, 512, generator=g).to(BF16).cuda(), picks(700, 32, 4, seed).cuda(), torch.rand(700, 4, generator=g).cuda(),
                (torch.randn(700, 512, generator=g) * 0.1).to(BF16).cuda()]

    def step(x, idx, wt, d):
        y, kept = ex.forward(x, idx, wt)
        dx, dw = ex.backward(d, kept)
        return (y, dx, dw) + tuning.add_rmsnorm_backward(r, w, dx, 1e-6, d_residual=d)

    batches = [inputs(s) for s in range(6)]
    alone = [step(*b) for b in batches]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, b in enumerate(batches):
        with torch.cuda.stream(sides[i % 2]):
            got.append(step(*b))
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(same_bits(s, t) for s, t in zip(a, b))
