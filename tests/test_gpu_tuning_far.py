"""Tuning calls whose buffers pass 2^32 elements: rows on both sides of that line against float64."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd.layer import MoERouter  # noqa: E402

U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32
FAR = 1 << 32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB")
    _lib.load()
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def rnd(*s, seed, std=1.0):
    """bf16 rows, made in pieces of 2^28 elements."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty(*s, dtype=BF16, device="cuda")
    for part in out.view(-1).split(1 << 28):
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda").mul_(std))
    return out


def close(got, ref, tol, what):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    bound = half * (ref.abs() + tol) + tol + 1e-37
    assert (err <= bound).all(), f"{what}: worst {(err / bound).max():.3g} of the bound"


def rows_at(T, width):
    """Rows at both ends and around the element number 2^31 and 2^32."""
    mid = [FAR // 2 // width, FAR // width]
    return torch.tensor(sorted({r for m in [0, T - 2, *mid] for r in range(m - 2, m + 2) if 0 <= r < T} | {T - 1})).cuda()


def test_adapters():
    T, K, N, R, G = FAR // 8192 + 333, 8192, 8192, 16, 3
    x, y = rnd(T, K, seed=1), rnd(T, N, seed=2)
    A, B = rnd(G, R, K, seed=3, std=K ** -0.5), rnd(G, N, R, seed=4, std=0.1)
    ad = (torch.arange(T, device="cuda") // 100 % (G + 1) - 1).to(torch.int32)
    l = tuning.LoRAAdapters(A, B)
    r = rows_at(T, K)
    before = y[r].clone()
    l.apply(x, ad, y)
    s = torch.stack([x[t].double() @ A[max(0, int(ad[t]))].double().t() for t in r]) * (ad[r] >= 0)[:, None]
    Bs = torch.stack([B[max(0, int(ad[t]))].double() for t in r])
    d = (Bs @ s[:, :, None])[:, :, 0]
    mag = (Bs.abs() @ torch.stack([x[t].double().abs() @ A[max(0, int(ad[t]))].double().abs().t() for t in r])[:, :, None])[:, :, 0]
    close(y[r], before.double() + d, mag * ((K + R + 16) * U + 2.0 ** -17), "y")
    # gradients: y in place of dy; only a few rows have an adapter, so that references stay small
    few = torch.full_like(ad, -1)
    few[r] = (torch.arange(len(r), device="cuda") % G).to(torch.int32)
    dy = y
    gx, ga, gb = l.backward(x, dy, few)
    for a in range(G):
        t = r[few[r] == a]
        X, D, Aa, Bb = x[t].double(), dy[t].double(), A[a].double(), B[a].double()
        u, si = D @ Bb, X @ Aa.t()
        um, sm = D.abs() @ Bb.abs(), X.abs() @ Aa.abs().t()
        close(gx[t], u @ Aa, (um @ Aa.abs()) * ((N + R + 16) * U + 2.0 ** -17), "dx")
        close(ga[a], u.t() @ X, (um.t() @ X.abs()) * (N + len(t) + 16) * U, "da")
        close(gb[a], D.t() @ si, (D.abs().t() @ sm) * (K + len(t) + 16) * U, "db")
    gx[r] = 0
    assert all(not bool(p.any()) for p in gx.split(1 << 15))


def test_combine():
    T, k, H = FAR // 8 // 4096 + 77, 8, 4096
    M = T * k
    Y, d = rnd(M, H, seed=5), rnd(T, H, seed=6)
    inv = torch.arange(M, device="cuda", dtype=torch.int32).flip(0).view(T, k).contiguous()
    w = torch.rand(T, k, device="cuda")
    r = rows_at(T, H * k)
    want_w = (Y[inv[r].long()].double() * d[r].double()[:, None]).sum(-1)
    mag = (Y[inv[r].long()].double() * d[r].double()[:, None]).abs().sum(-1)
    dY, dw = tuning.unpermute_backward(d, Y, inv, w, dY=Y)
    close(dw[r], want_w, mag * (H + 2) * U, "d weight")
    close(dY[inv[r].long()], w[r].to(BF16).double()[:, :, None] * d[r].double()[:, None], 0.0, "dY")


def test_router_rows():
    E, k = 512, 2
    T = FAR // E + 1001
    lg = rnd(T, E, seed=7)
    idx = (torch.arange(T * k, device="cuda") % E).to(torch.int32).view(T, k)
    mask = torch.zeros(T, dtype=torch.bool, device="cuda")
    r = rows_at(T, E)
    mask[r] = True
    router = MoERouter(E, k)
    b = tuning.balance_loss(router, lg, idx, mask=mask)
    n, s = len(r), lg[r].double()
    counts = torch.bincount(idx[r].flatten().long(), minlength=E)
    assert torch.equal(b.counts[:-1].long(), counts) and int(b.counts[-1]) == n
    P = torch.softmax(s, 1).sum(0)
    close(b.prob_sum, P, P * (E + n + 24) * U, "P")
    dw = torch.randn(T, k, device="cuda")
    got = tuning.router_backward(router, lg, idx, dw, mask=mask)
    at = idx[r].long()
    w, g = torch.softmax(s.gather(1, at), 1), dw[r].double()
    want = torch.zeros(n, E, dtype=torch.float64, device="cuda").scatter_add(1, at, w * (g - (g * w).sum(1, keepdim=True)))
    close(got[r], want, 2 * g.abs().sum(1, keepdim=True).expand(n, E) * (k + 24) * U, "d logits")
    got[r] = 0
    assert all(not bool(p.any()) for p in got.split(1 << 19))
