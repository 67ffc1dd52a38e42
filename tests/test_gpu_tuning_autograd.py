"""Tuning calls beside autograd: writes into tensors that it saved are noticed, and the calls serve as the body of a
torch.autograd.Function."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd.layer import MoERouter  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    _lib.load()
    yield
    torch.cuda.synchronize()


def rnd(*s, seed=0):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed)).cuda()


def adapters(G=2, R=8, K=32, N=24):
    return tuning.LoRAAdapters(rnd(G, R, K, seed=1) * K ** -0.5, rnd(G, N, R, seed=2), torch.tensor([1.0, 0.5]).cuda())


def test_writes_count_as_changes_in_place():
    """Each tensor of the caller's that a call writes has its version raised, and no other."""
    l, x, ad = adapters(), rnd(5, 32, seed=3), torch.tensor([0, 1, -1, 0, 1], dtype=torch.int32).cuda()
    y, dy, dx = rnd(5, 24, seed=4), rnd(5, 24, seed=5), rnd(5, 32, seed=6)
    lg, idx, out = rnd(5, 8), torch.arange(10, dtype=torch.int32).reshape(5, 2).cuda() % 8, torch.empty(5, 8).cuda()
    Y, inv, w = rnd(10, 8), torch.arange(10, dtype=torch.int32).cuda(), rnd(5, 2)
    o2, dx2, g = torch.empty_like(y), torch.empty_like(dx), rnd(5, 8)
    held = dict(l_a=l.a, l_b=l.b, x=x, ad=ad, y=y, dy=dy, dx=dx, lg=lg, idx=idx, out=out, Y=Y, inv=inv, w=w, o2=o2, dx2=dx2, g=g)
    for call, written in [
            (lambda: l.apply(x, ad, y), "y"), (lambda: l.apply(x, ad, y, out=o2), "o2"), (lambda: l.apply(x, ad), None),
            (lambda: l.backward(x, dy, ad, dx=dx), "dx"), (lambda: l.backward(x, dy, ad, dx=dx, dx_out=dx2), "dx2"),
            (lambda: l.backward(x, dy, ad), None), (lambda: l.backward(x, dy, ad, need_dx=False), None),
            (lambda: tuning.router_backward(MoERouter(8, 2), lg, idx, w, out=out), "out"),
            (lambda: tuning.router_backward(MoERouter(8, 2), lg, idx, w), None),
            (lambda: tuning.unpermute_backward(g, Y, inv, w, dY=Y), "Y"), (lambda: tuning.unpermute_backward(g, Y, inv, w), None)]:
        before = {k: t._version for k, t in held.items()}
        call()
        raised = [k for k, t in held.items() if t._version != before[k]]
        assert raised == ([] if written is None else [written])


def test_a_saved_tensor_that_adapters_write_is_noticed():
    l, x, ad, y = adapters(), rnd(5, 32), torch.zeros(5, dtype=torch.int32).cuda(), rnd(5, 24)
    w = torch.ones(5, 24, device="cuda", requires_grad=True)
    z = (w * y).sum()  # saves y
    l.apply(x, ad, y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_inference_mode():
    l, x, ad = adapters(), rnd(5, 32), torch.zeros(5, dtype=torch.int32).cuda()
    want = l.apply(x, ad)
    with torch.inference_mode():
        y = torch.zeros(5, 24, device="cuda")
        assert torch.equal(l.apply(x, ad, y), want) and torch.equal(y, want)


class Adapted(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, scale, ad, y):
        ctx.save_for_backward(x, a, b, scale, ad)
        return tuning.LoRAAdapters(a, b, scale).apply(x, ad, y, out=torch.empty_like(y))

    @staticmethod
    def backward(ctx, dy):
        x, a, b, scale, ad = ctx.saved_tensors
        dx, da, db = tuning.LoRAAdapters(a, b, scale).backward(x, dy.contiguous(), ad)
        return dx, da, db, None, None, dy


def test_the_body_of_an_autograd_function():
    """Leaves that require gradients go through a Function made of the calls; its gradients are the formula's in float64."""
    l, x, ad, y = adapters(), rnd(9, 32), (torch.arange(9) % 3 - 1).to(torch.int32).cuda(), rnd(9, 24)
    leaves = [t.clone().requires_grad_(True) for t in (x, l.a, l.b, y)]
    out = Adapted.apply(leaves[0], leaves[1], leaves[2], l.scale, ad, leaves[3])
    (out * out).sum().backward()
    ref = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    i = ad.long().cpu()
    s = torch.where(i < 0, 0.0, l.scale.double().cpu()[i.clamp(min=0)])
    A, B = ref[1][i.clamp(min=0)], ref[2][i.clamp(min=0)]
    o = ref[3] + s[:, None] * (B @ (A @ ref[0][:, :, None]))[:, :, 0]
    (o * o).sum().backward()
    assert (out.detach().double().cpu() - o.detach()).abs().max() <= 1e-5 * o.detach().abs().max()
    for got, want in zip(leaves, ref):
        # sums of up to 32 + 8 + 9 + 24 products in fp32, of magnitudes up to a few hundred times the largest gradient's share
        assert (got.grad.double().cpu() - want.grad).abs().max() <= 1e-5 * want.grad.abs().max()
