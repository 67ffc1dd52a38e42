"""Adapter gradients over the ways that rows spread over adapters: partial gradients that fill their workspace, and the
plans that list many rows. References and bounds in float64: a result rounded to type t is off by eps(t)/2 of its value, a
sum of n fp32 products by (n + c) 2^-24 of the sum of their magnitudes, a factor kept as two 16-bit parts by 2^-17."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd._lib import check  # noqa: E402
from ffai_amd.layer import moe_dtype  # noqa: E402

U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    _lib.load()
    yield
    torch.cuda.synchronize()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def close(got, ref, tol, what):
    half = torch.finfo(got.dtype).eps / 2
    low = torch.finfo(got.dtype).smallest_normal * half
    got, ref = got.double().cpu(), ref.double().cpu()
    err = (got - ref).abs()
    bound = half * (ref.abs() + tol) + tol + low + torch.finfo(torch.float32).tiny
    assert (err <= bound).all(), f"{what}: {int((~(err <= bound)).sum())} off, worst {(err / bound).max():.3g} of the bound"


def inputs(T, K, N, R, G, dt, seed):
    g = gen(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return (rnd(T, K).to(dt), (rnd(G, R, K) * K ** -0.5).to(dt), (rnd(G, N, R) * 0.1).to(dt),
            torch.rand(G, generator=g) + 0.5, rnd(T, N).to(dt))


def check_gradients(got, x, A, B, scale, ad, dy, adapters):
    """(dx, da, db) of the given adapters, and of rows without one."""
    gx, ga, gb = (t.cpu() for t in got)
    K, N, R = x.shape[1], B.shape[1], A.shape[1]
    sp = 0.0 if x.dtype == F32 else 2.0 ** -17
    for a in adapters:
        r = (ad == a).nonzero()[:, 0]
        if not len(r):
            assert (ga[a] == 0).all() and (gb[a] == 0).all()
            continue
        s, X, D, Aa, Bb = float(scale[a]), x[r].double(), dy[r].double(), A[a].double(), B[a].double()
        u, s1 = s * D @ Bb, s * X @ Aa.t()
        um, sm = s * D.abs() @ Bb.abs(), s * X.abs() @ Aa.abs().t()
        close(gx[r], u @ Aa, (um @ Aa.abs()) * ((N + R + 16) * U + sp), f"dx {a}")
        close(ga[a], u.t() @ X, (um.t() @ X.abs()) * ((N + len(r) + 16) * U + sp), f"da {a}")
        close(gb[a], D.t() @ s1, (D.abs().t() @ sm) * ((K + len(r) + 16) * U + sp), f"db {a}")
    none = (ad < 0) | (ad >= A.shape[0])
    assert (gx[none] == 0).all()


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("rows,K,N,R", [
    ([65] * 10, 64, 64, 8),                                          # every adapter one chunk of 64 rows and one row more
    ([200, 0, 1, 200, 64, 200, 30], 2048, 2048, 64),                 # several, one and no chunk in turn
    ([65] + [1] * 70 + [130, 0, 0, 65] + [64] * 60 + [66], 72, 136, 24),   # past the first 64 adapters
    ([64] * 12, 64, 64, 16), ([1000], 136, 72, 40),
])
def test_gradients_of_chunks_in_a_workspace_of_its_size(dt, rows, K, N, R):
    T, G = sum(rows), len(rows)
    ad = torch.repeat_interleave(torch.arange(G), torch.tensor(rows))
    ad = ad[torch.randperm(T, generator=gen(3))].to(torch.int32)
    x, A, B, scale, dy = inputs(T, K, N, R, G, dt, T + R)
    dev = [t.cuda() for t in (x, A, B, scale, ad, dy)]
    xc, Ac, Bc, sc, ac, dc = dev
    lib = _lib.load()
    desc = _lib.Lora(Ac.data_ptr(), Bc.data_ptr(), sc.data_ptr(), moe_dtype(dt), R, N, K, G)
    need = lib.moe_lora_backward_workspace_bytes(C.byref(desc), T)
    ws = torch.full((need + 65536,), 255, dtype=torch.uint8, device="cuda")
    out = [torch.full_like(t, 9.0) for t in (xc, Ac, Bc)]
    check(lib.moe_lora_backward(C.byref(desc), xc.data_ptr(), dc.data_ptr(), T, ac.data_ptr(), None,
                                *(o.data_ptr() for o in out), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (ws[need:] == 255).all()
    check_gradients(out, x, A, B, scale, ad, dy, range(G))
    for a, b in zip(out, tuning.LoRAAdapters(Ac, Bc, sc).backward(xc, dc, ac)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("T,G,spread", [
    (16384, 1, "some"), (16385, 1, "some"), (20011, 1, "some"), (20011, 2, "even"), (17001, 300, "even"), (33001, 70, "most"),
    (33001, 1024, "even"), (20011, 5, "none"), (40000, 3, "last"),
])
def test_gradients_of_more_rows_than_a_launch_lists(dt, T, G, spread):
    """The plans of many rows: a block per adapter, and chunks of rows with their own counts where there are few
    adapters, or many, or more rows still. Ids out of range among them."""
    K, N, R = 24, 40, 16
    x, A, B, scale, dy = inputs(T, K, N, R, G, dt, T + G)
    g = gen(G)
    ad = torch.randint(-1, G + 1, (T,), generator=g)
    if spread == "most":
        ad = torch.where(torch.rand(T, generator=g) < 0.6, 3, ad)
    elif spread == "none":
        ad = torch.where(torch.rand(T, generator=g) < 0.5, -1, 1 << 30)
    elif spread == "last":
        ad = torch.where(torch.arange(T) < T - 7, -5, G - 1)
    ad = ad.to(torch.int32)
    l = tuning.LoRAAdapters(A.cuda(), B.cuda(), scale.cuda())
    dev = x.cuda(), dy.cuda(), ad.cuda()
    got = l.backward(*dev)
    check_gradients(got, x, A, B, scale, ad, dy, range(G) if G <= 5 else [0, 1, 3, 62, 63, 64, 65, G - 2, G - 1])
    for a, b in zip(got, l.backward(*dev)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
