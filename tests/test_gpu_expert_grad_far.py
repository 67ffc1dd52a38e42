"""Gradients through the experts with buffers that pass 2^32 bytes or elements: rows on both sides of those lines
against float64."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_expert_grad import stack  # noqa: E402
from test_gpu_tuning_far import BF16, F32, FAR, U, close, rnd, rows_at  # noqa: E402

from ffai_amd import _lib, tuning  # noqa: E402


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


@pytest.mark.parametrize("T,N,K,gather", [
    (FAR // 4096 + 777, 2560, 64, True),     # gathered rows of 5.4 GB, blocks of 256 rows
    (4200, 1 << 20, 32, True),               # rows of 2 MB each, 8.8 GB, blocks of 128 rows
    (FAR // 4096 + 777, 64, 2560, False),    # a result of 5.4 GB
])
def test_products(T, N, K, gather):
    E = 2 if T > 5000 else 1
    p, W = stack(E, N, K, 4, 32, BF16, 5)
    W = W.cuda()
    dy = rnd(T, N, seed=1, std=0.01)
    cut = T // 3 if E == 2 else T
    offsets = torch.tensor([0, cut, T][:E + 1] if E == 2 else [0, T], dtype=torch.int32).cuda()
    perm = torch.randperm(T, generator=torch.Generator().manual_seed(3)).to(torch.int32).cuda() if gather else None
    dx = tuning.expert_matmul_backward(p, dy, offsets, perm=perm, top_k=1)
    at = rows_at(T, max(N, K))
    if gather:  # positions of the farthest rows as well
        at = torch.unique(torch.cat([at, perm.argsort()[at]]))
    row = perm[at].long() if gather else at
    e = (at >= cut).long() if E == 2 else torch.zeros_like(at)
    for r, q, x in zip(row.tolist(), at.tolist(), e.tolist()):
        d = dy[r].double()
        ref, mag = d @ W[x], d.abs() @ W[x].abs()
        close(dx[q], ref, mag * (2.0 ** -8 + (N + 8) * U), f"row {q}")


def test_activation():
    M, n = FAR // 2048 + 333, 2080
    dt = BF16
    gate, up = rnd(M, n, seed=1), rnd(M, n, seed=2)
    h, kept = tuning.activation_save(gate, up)
    at = rows_at(M, n)
    g, u = gate[at].double(), up[at].double()
    ref = g * torch.sigmoid(g) * u
    close(h[at], ref, ref.abs() * 64 * U, "h")
    del h, gate, up
    step = torch.exp2(kept.scales[:, at].double() - 133).repeat_interleave(32, 2)
    v = kept.codes[:, at].double() * step
    assert ((v - torch.stack([g, u])).abs() <= step / 2).all()
    back = kept.restore(dt)
    assert torch.equal(back[:, at].double(), v)
    del back
    dh = rnd(M, n, seed=3, std=0.01)
    w = torch.rand(M, device="cuda")
    perm = torch.arange(M - 1, -1, -1, device="cuda", dtype=torch.int32)
    got = tuning.activation_backward(kept, dh, topk_weight=w, perm=perm)
    pick = perm[at].long()
    d, r, s = dh[at].double(), w[pick].to(dt).double()[:, None], torch.sigmoid(v[0])
    close(got.d_up[at], r * d * v[0] * s, (r * d * v[0]).abs() * 64 * U, "d_up")
    slope = (s + v[0] * s * (1 - s)) * v[1]
    close(got.d_gate[at], r * d * slope, (r * d).abs() * (slope.abs() + v[1].abs() * (1 + v[0].abs())) * 64 * U, "d_gate")
    hv = v[0] * s * v[1]
    close(got.d_weight[pick], (d * hv).sum(1), (d * hv).abs().sum(1) * (n + 64) * U, "d_weight")


def test_rows_back_and_norm():
    T, H = FAR // 4096 + 99, 4104
    dX = rnd(T, H, seed=1)
    inv = torch.randperm(T, generator=torch.Generator().manual_seed(4)).to(torch.int32).cuda()[:, None]
    dx = tuning.permute_backward(dX, inv.contiguous())
    at = rows_at(T, H)
    at = torch.unique(torch.cat([at, inv[:, 0].argsort()[at]]))
    assert torch.equal(dx[at], dX[inv[at, 0].long()])
    del dX
    w, dn, eps = (1 + 0.1 * torch.randn(H, device="cuda")).to(BF16), rnd(T, H, seed=2, std=0.01), 1e-6
    din, dw = tuning.add_rmsnorm_backward(dx, w, dn, eps)
    x, d, W = dx[at].double(), dn[at].double(), w.double()
    s = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    q, p = x * s, d * W
    m = (p * q).mean(1, keepdim=True)
    close(din[at], s * (p - q * m), s * (p.abs() + q.abs() * m.abs() + q.abs() * (p * q).abs().mean(1, keepdim=True)) * (H + 64) * U, "d_in")
    # the weight's gradient, of all rows, in pieces
    ref, mag = torch.zeros(H, dtype=torch.float64, device="cuda"), torch.zeros(H, dtype=torch.float64, device="cuda")
    for a, b in zip(dx.split(1 << 15), dn.split(1 << 15)):
        a, b = a.double(), b.double()
        t = b * a / torch.sqrt((a * a).mean(1, keepdim=True) + eps)
        ref += t.sum(0)
        mag += t.abs().sum(0)
    # a block's rows one after another, then the blocks'
    close(dw, ref, mag * (T / 512 + 512 + H / 2 + 64) * U, "d_weight")
