"""Refusals of the tuning entry points: contract violations are rejected on
the host, before any launch, through the C ABI and through ffai_amd.tuning."""
import ctypes as C

import pytest

from ffai_amd import _lib
from ffai_amd._lib import MOE_BF16, MOE_ERR_INVALID, MOE_ERR_UNSUPPORTED, MOE_ERR_WORKSPACE, MOE_OK, Lora

torch = pytest.importorskip("torch")

from ffai_amd import tuning  # noqa: E402
from ffai_amd.layer import MoEGatingMode, MoERouter  # noqa: E402

BIG = 1 << 40


def p(i):
    """A distinct, 16-byte aligned address that nothing reads."""
    return C.c_void_p(BIG * (i + 1))


BAL = dict(logits=p(0), dtype=MOE_BF16, T=64, E=32, k=4, gating=0, ls=1.0, idx=p(1), mask=None, counts=p(2),
           P=p(3), losses=p(4), ws=None, ws_bytes=0)
RB = dict(logits=p(0), dtype=MOE_BF16, T=64, E=32, k=4, gating=0, norm=1, eb=None, ls=1.0, rs=1.0, es=None,
          idx=p(1), dw=p(2), counts=p(3), bal=0.1, z=0.0, mask=None, out=p(4))
UB = dict(g=p(0), Y=p(1), inv=p(2), w=p(3), T=4, H=64, k=2, dY=p(4), dw=p(5), dtype=MOE_BF16)


def call(fn, base, **kw):
    return getattr(_lib.load(), fn)(*{**base, **kw}.values(), None)


BAD_ROWS = [
    (dict(T=0), MOE_ERR_INVALID, "T must be positive"), (dict(T=-3), MOE_ERR_INVALID, "T must be positive"),
    (dict(E=0), MOE_ERR_INVALID, "nExperts"), (dict(k=0), MOE_ERR_INVALID, "topK"),
    (dict(k=33), MOE_ERR_INVALID, "topK"), (dict(E=513), MOE_ERR_UNSUPPORTED, "above 512"),
    (dict(E=128, k=65), MOE_ERR_UNSUPPORTED, "above 64"), (dict(dtype=3), MOE_ERR_INVALID, "dtype"),
    (dict(gating=3), MOE_ERR_INVALID, "gating"), (dict(ls=float("nan")), MOE_ERR_INVALID, "finite"),
    (dict(T=1 << 30), MOE_ERR_INVALID, "too large"), (dict(logits=None), MOE_ERR_INVALID, "NULL"),
    (dict(idx=None), MOE_ERR_INVALID, "NULL"),
]


@pytest.mark.parametrize("kw,status,needle", BAD_ROWS + [
    (dict(counts=None), MOE_ERR_INVALID, "NULL"), (dict(P=None), MOE_ERR_INVALID, "NULL"),
    (dict(losses=None), MOE_ERR_INVALID, "NULL"),
    (dict(T=100000), MOE_ERR_WORKSPACE, "workspace"),
    (dict(T=100000, ws=p(6), ws_bytes=16), MOE_ERR_WORKSPACE, "workspace"),
    (dict(T=100000, ws=C.c_void_p(BIG * 7 + 8), ws_bytes=BIG), MOE_ERR_WORKSPACE, "aligned"),
])
def test_balance_loss_refuses(kw, status, needle):
    assert call("moe_balance_loss", BAL, **kw) == status
    assert needle in _lib.last_error()


@pytest.mark.parametrize("kw,status,needle", BAD_ROWS + [
    (dict(out=None), MOE_ERR_INVALID, "NULL"), (dict(rs=float("inf")), MOE_ERR_INVALID, "finite"),
    (dict(bal=float("nan")), MOE_ERR_INVALID, "coefficients"), (dict(z=float("inf")), MOE_ERR_INVALID, "coefficients"),
    (dict(counts=None), MOE_ERR_INVALID, "counts"), (dict(counts=None, bal=0.0, z=1e-3), MOE_ERR_INVALID, "counts"),
    (dict(out=p(0)), MOE_ERR_INVALID, "overlaps"), (dict(out=C.c_void_p(BIG + 64 * 32 * 2 - 2)), MOE_ERR_INVALID, "overlaps"),
])
def test_router_backward_refuses(kw, status, needle):
    assert call("moe_router_backward", RB, **kw) == status
    assert needle in _lib.last_error()


@pytest.mark.parametrize("kw,status,needle", [
    (dict(g=None), MOE_ERR_INVALID, "NULL"), (dict(Y=None), MOE_ERR_INVALID, "NULL"),
    (dict(inv=None), MOE_ERR_INVALID, "NULL"), (dict(w=None), MOE_ERR_INVALID, "NULL"),
    (dict(dw=None), MOE_ERR_INVALID, "NULL"), (dict(T=0), MOE_ERR_INVALID, "positive"),
    (dict(H=0), MOE_ERR_INVALID, "positive"), (dict(k=0), MOE_ERR_INVALID, "positive"),
    (dict(H=60), MOE_ERR_UNSUPPORTED, "multiple of 8"), (dict(dtype=7), MOE_ERR_INVALID, "dtype"),
    (dict(T=1 << 30, k=2), MOE_ERR_INVALID, "too large"),
    (dict(Y=C.c_void_p(BIG + 8)), MOE_ERR_INVALID, "aligned"), (dict(g=C.c_void_p(BIG + 2)), MOE_ERR_INVALID, "aligned"),
    (dict(dY=C.c_void_p(BIG * 2 + 16)), MOE_ERR_INVALID, "overlaps"),
    (dict(dY=C.c_void_p(BIG + 256)), MOE_ERR_INVALID, "overlaps"),
])
def test_unpermute_backward_refuses(kw, status, needle):
    assert call("moe_unpermute_backward", UB, **kw) == status
    assert needle in _lib.last_error()


def lora(**kw):
    f = dict(a=BIG * 21, b=BIG * 22, scale=BIG * 23, dtype=MOE_BF16, rank=16, n=64, k=128, n_adapters=4)
    f.update(kw)
    return Lora(*f.values())


BAD_LORA = [
    (dict(a=None), MOE_ERR_INVALID, "non-NULL"), (dict(b=None), MOE_ERR_INVALID, "non-NULL"),
    (dict(a=BIG + 8), MOE_ERR_INVALID, "aligned"), (dict(scale=BIG + 2), MOE_ERR_INVALID, "aligned"),
    (dict(dtype=5), MOE_ERR_INVALID, "dtype"), (dict(rank=0), MOE_ERR_INVALID, "positive"),
    (dict(n_adapters=0), MOE_ERR_INVALID, "positive"), (dict(rank=12), MOE_ERR_UNSUPPORTED, "multiples of 8"),
    (dict(n=60), MOE_ERR_UNSUPPORTED, "multiples of 8"), (dict(k=4), MOE_ERR_UNSUPPORTED, "multiples of 8"),
    (dict(rank=136), MOE_ERR_UNSUPPORTED, "above 128"), (dict(n=(1 << 20) + 8), MOE_ERR_UNSUPPORTED, "2^20"),
]


@pytest.mark.parametrize("kw,status,needle", BAD_LORA)
def test_lora_descriptor_refused(kw, status, needle):
    lib, l = _lib.load(), lora(**kw)
    calls = [lambda: lib.moe_validate_lora(C.byref(l)),
             lambda: lib.moe_lora_apply(C.byref(l), p(0), 4, p(1), p(2), p(3), p(4), BIG, None),
             lambda: lib.moe_lora_backward(C.byref(l), p(0), p(1), 4, p(2), p(3), p(4), p(5), p(6), p(7), BIG, None)]
    for c in calls:
        assert c() == status
        assert needle in _lib.last_error()
    assert lib.moe_lora_workspace_bytes(C.byref(l), 4) == 0
    assert lib.moe_lora_backward_workspace_bytes(C.byref(l), 4) == 0


APPLY = dict(x=p(0), T=4, ad=p(1), yin=p(2), y=p(3), ws=p(4), ws_bytes=BIG)
BACK = dict(x=p(0), dy=p(1), T=4, ad=p(2), dxin=p(3), dx=p(4), da=p(5), db=p(6), ws=p(7), ws_bytes=BIG)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(x=None), MOE_ERR_INVALID, "NULL"), (dict(ad=None), MOE_ERR_INVALID, "NULL"),
    (dict(y=None), MOE_ERR_INVALID, "NULL"), (dict(T=0), MOE_ERR_INVALID, "positive"),
    (dict(x=C.c_void_p(BIG + 4)), MOE_ERR_INVALID, "aligned"), (dict(yin=C.c_void_p(BIG + 4)), MOE_ERR_INVALID, "aligned"),
    (dict(y=p(0)), MOE_ERR_INVALID, "overlaps x"), (dict(yin=C.c_void_p(BIG * 4 + 16)), MOE_ERR_INVALID, "y_in"),
    (dict(ws=None), MOE_ERR_WORKSPACE, "workspace"), (dict(ws_bytes=15), MOE_ERR_WORKSPACE, "workspace"),
    (dict(ws=C.c_void_p(BIG * 5 + 4)), MOE_ERR_WORKSPACE, "aligned"),
])
def test_lora_apply_refuses(kw, status, needle):
    l = lora(n=4096, k=4096, rank=64)  # large enough that a few rows need a workspace
    assert _lib.load().moe_lora_apply(C.byref(l), *{**APPLY, **kw}.values(), None) == status
    assert needle in _lib.last_error()


@pytest.mark.parametrize("kw,status,needle", [
    (dict(x=None), MOE_ERR_INVALID, "NULL"), (dict(dy=None), MOE_ERR_INVALID, "NULL"),
    (dict(ad=None), MOE_ERR_INVALID, "NULL"), (dict(T=-1), MOE_ERR_INVALID, "positive"),
    (dict(dxin=None, dx=None, da=None, db=None), MOE_ERR_INVALID, "no gradient"),
    (dict(dx=None), MOE_ERR_INVALID, "dx_in without dx"), (dict(da=C.c_void_p(BIG + 8)), MOE_ERR_INVALID, "aligned"),
    (dict(dx=p(0)), MOE_ERR_INVALID, "overlaps"), (dict(dx=p(1)), MOE_ERR_INVALID, "overlaps"),
    (dict(dx=C.c_void_p(BIG * 4 + 32)), MOE_ERR_INVALID, "overlaps"),
    (dict(ws_bytes=1024), MOE_ERR_WORKSPACE, "workspace"), (dict(ws=None), MOE_ERR_WORKSPACE, "workspace"),
])
def test_lora_backward_refuses(kw, status, needle):
    l = lora()
    assert _lib.load().moe_lora_backward(C.byref(l), *{**BACK, **kw}.values(), None) == status
    assert needle in _lib.last_error()


def test_lora_backward_refuses_many_adapters():
    l = lora(n_adapters=1025)
    lib = _lib.load()
    assert lib.moe_validate_lora(C.byref(l)) == MOE_OK
    assert lib.moe_lora_backward(C.byref(l), *BACK.values(), None) == MOE_ERR_UNSUPPORTED
    assert "1024" in _lib.last_error()


def test_workspace_sizes():
    """Workspaces grow with the rows; a few rows of a balance loss and small
    adapters need none."""
    lib, l = _lib.load(), lora(n=4096, k=4096, rank=64)
    small = lora()
    assert [lib.moe_lora_workspace_bytes(C.byref(small), T) for T in (1, 100, 10000)] == [0, 0, 0]
    assert lib.moe_balance_loss_workspace_bytes(1, 32) == 0
    assert lib.moe_balance_loss_workspace_bytes(65536, 256) > 0
    assert lib.moe_balance_loss_workspace_bytes(0, 32) == lib.moe_balance_loss_workspace_bytes(8, 513) == 0
    for f in (lib.moe_lora_workspace_bytes, lib.moe_lora_backward_workspace_bytes):
        assert 0 < f(C.byref(l), 1) <= f(C.byref(l), 100) <= f(C.byref(l), 10000)
        assert f(C.byref(l), 0) == 0
        for G in (1, 3, 40):
            g = lora(n_adapters=G, n=4096, k=4096, rank=64)
            sizes = [f(C.byref(g), T) for T in list(range(1, 700)) + [1000, 4096, 40000]]
            assert sizes == sorted(sizes)
            g = lora(n_adapters=G, n=64, k=64, rank=8)  # its gradients are cut into many chunks
            sizes = [f(C.byref(g), T) for T in range(1, 40000, 7)]
            assert sizes == sorted(sizes)
    for E in (1, 32, 129, 512):
        sizes = [lib.moe_balance_loss_workspace_bytes(T, E) for T in range(1, 40000, 11)]
        assert sizes == sorted(sizes)


# ------------------------------------------------------------- Python side --

def test_python_refuses_host_tensors():
    r = MoERouter(8, 2)
    lg, idx = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="on a GPU"):
        tuning.balance_loss(r, lg, idx)
    with pytest.raises(ValueError, match="on a GPU"):
        tuning.router_backward(r, lg, idx)
    with pytest.raises(ValueError, match="on a GPU"):
        tuning.unpermute_backward(torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8, dtype=torch.int32),
                                  torch.zeros(4, 2))


@pytest.mark.parametrize("kw,needle", [
    (dict(logits=torch.zeros(4, 9)), r"logits must be \[4, 8\]"),
    (dict(logits=torch.zeros(0, 8)), "must have rows"),
    (dict(logits=torch.zeros(4, 8, dtype=torch.float64)), "dtype"),
    (dict(logits=torch.zeros(8, 4).t()), "contiguous"),
    (dict(topk_idx=torch.zeros(4, 2, dtype=torch.int64)), "dtype"),
    (dict(topk_idx=torch.zeros(4, 3, dtype=torch.int32)), "topk_idx must be"),
    (dict(mask=torch.ones(5, dtype=torch.bool)), "mask must be"),
    (dict(mask=torch.ones(4)), "mask dtype"),
])
def test_python_router_refusals(kw, needle):
    base = dict(logits=torch.zeros(4, 8), topk_idx=torch.zeros(4, 2, dtype=torch.int32))
    for f in (tuning.balance_loss, tuning.router_backward):
        with pytest.raises(ValueError, match=needle):
            f(MoERouter(8, 2, MoEGatingMode.softmaxThenTopK), **{**base, **kw})


@pytest.mark.parametrize("a,b,scale,needle", [
    (torch.zeros(2, 8), torch.zeros(2, 8, 8), None, "3 dimensions"),
    (torch.zeros(2, 8, 16), torch.zeros(3, 8, 8), None, "b must be"),
    (torch.zeros(2, 8, 16), torch.zeros(2, 8, 8, dtype=torch.float16), None, "b dtype"),
    (torch.zeros(2, 8, 16), torch.zeros(2, 8, 8), torch.ones(3), "scale must be"),
    (torch.zeros(2, 8, 16), torch.zeros(2, 8, 8), torch.ones(2, dtype=torch.float64), "scale dtype"),
    (torch.zeros(2, 16, 8).transpose(1, 2), torch.zeros(2, 8, 8), None, "contiguous"),
])
def test_python_lora_refusals(a, b, scale, needle):
    with pytest.raises(ValueError, match=needle):
        tuning.LoRAAdapters(a, b, scale)


def test_python_lora_rank_refused_by_the_library():
    with pytest.raises(_lib.MoeError, match="multiples of 8"):
        tuning.LoRAAdapters(torch.zeros(2, 12, 16), torch.zeros(2, 8, 12))


def test_python_lora_call_refusals():
    l = tuning.LoRAAdapters(torch.zeros(2, 8, 16), torch.zeros(2, 24, 8))
    x, ad, y, dy = torch.zeros(3, 16), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 24), torch.zeros(3, 24)
    for bad, needle in [(lambda: l.apply(torch.zeros(3, 8), ad, y), "x must be"),
                        (lambda: l.apply(x, ad.long(), y), "adapter dtype"),
                        (lambda: l.apply(x, ad[:2], y), "adapter must be"),
                        (lambda: l.apply(x, ad, torch.zeros(3, 16)), "y must be"),
                        (lambda: l.apply(x, ad, y, out=torch.zeros(2, 24)), "out must be"),
                        (lambda: l.apply(x, ad, y), "on a GPU"),
                        (lambda: l.backward(x, y.half(), ad), "dy dtype"),
                        (lambda: l.backward(x, dy, ad, dx=torch.zeros(3, 24)), "dx must be"),
                        (lambda: l.backward(x, dy, ad, dx=x, need_dx=False), "need_dx"),
                        (lambda: l.backward(x, dy, ad), "on a GPU")]:
        with pytest.raises(ValueError, match=needle):
            bad()


@pytest.mark.parametrize("T", [(1 << 23) + 1, (1 << 31) - 1])
def test_rows_past_a_launch_refused(T):
    lib, l = _lib.load(), lora(n=8, k=8, rank=8)
    far = BIG << 6  # buffers of so many rows stay apart
    at = [C.c_void_p(far * (i + 1)) for i in range(8)]
    assert lib.moe_lora_apply(C.byref(l), at[0], T, at[1], at[2], at[3], None, 0, None) == MOE_ERR_UNSUPPORTED
    assert "T above" in _lib.last_error()
    assert lib.moe_lora_backward(C.byref(l), at[0], at[1], T, at[2], at[3], at[4], at[5], at[6], at[7], far,
                                 None) == MOE_ERR_UNSUPPORTED
    assert "T above" in _lib.last_error()
    assert lib.moe_lora_workspace_bytes(C.byref(l), T) == lib.moe_lora_backward_workspace_bytes(C.byref(l), T) == 0
    assert call("moe_unpermute_backward", UB, T=T, k=1, H=8) == MOE_ERR_UNSUPPORTED
    assert "T above" in _lib.last_error()


A, B = C.c_void_p(BIG * 21), C.c_void_p(BIG * 22 + 64)


@pytest.mark.parametrize("kw,needle", [
    (dict(da=p(0)), "input"), (dict(db=p(1)), "input"), (dict(da=p(3)), "input"), (dict(db=p(4)), "gradients overlap"),
    (dict(da=p(6)), "gradients overlap"), (dict(da=A), "adapters"), (dict(db=B), "adapters"), (dict(dx=B), "adapters"),
    (dict(dx=A), "adapters"), (dict(dx=None, dxin=None, db=p(5)), "gradients overlap"),
])
def test_lora_backward_refuses_overlaps(kw, needle):
    l = lora()
    assert _lib.load().moe_lora_backward(C.byref(l), *{**BACK, **kw}.values(), None) == MOE_ERR_INVALID
    assert needle in _lib.last_error()


@pytest.mark.parametrize("y", [A, B])
def test_lora_apply_refuses_writing_adapters(y):
    l = lora()
    assert _lib.load().moe_lora_apply(C.byref(l), *{**APPLY, "y": y, "yin": None}.values(), None) == MOE_ERR_INVALID
    assert "overlaps the adapters" in _lib.last_error()


def test_python_unpermute_backward_inv_perm():
    g, Y, w = torch.zeros(3, 8), torch.zeros(6, 8), torch.zeros(3, 2)
    for bad in ([0] * 6, torch.zeros(7, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="inv_perm must be"):
            tuning.unpermute_backward(g, Y, bad, w)


def test_python_lora_memory_checked_each_call():
    """A tensor whose memory is set to rows that lie apart is refused, also where
    its address, shape and type stay."""
    wide = torch.zeros(4, 8, 16)
    l = tuning.LoRAAdapters(wide[:2], torch.zeros(2, 24, 8))
    x, ad = torch.zeros(3, 16), torch.zeros(3, dtype=torch.int32)
    l.a.data = wide[::2]
    with pytest.raises(ValueError, match="a must be contiguous"):
        l.apply(x, ad)
    assert l == l and l != tuning.LoRAAdapters(l.b, torch.zeros(2, 16, 24))
