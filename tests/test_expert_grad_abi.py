"""Refusals of the calls that take gradients through the quantised experts:
contract violations are rejected on the host, before any launch."""
import ctypes as C

import pytest

from ffai_amd import _lib
from ffai_amd._lib import MOE_BF16, MOE_ERR_INVALID, MOE_ERR_UNSUPPORTED, MOE_ERR_WORKSPACE, MOE_F32, QProj

BIG = 1 << 44


def p(i, off=0):
    """A distinct, 16-byte aligned address that nothing reads."""
    return C.c_void_p(BIG * (i + 1) + off)


def proj(**kw):
    f = dict(weight=p(20), scales=p(21), biases=p(22), out_bias=None, bits=4, group_size=64, sb_dtype=MOE_BF16, n=128, k=256,
             n_experts=8)
    f.update(kw)
    return C.byref(QProj(*f.values()))


def other(**kw):
    return proj(**{**dict(weight=p(23), scales=p(24), biases=p(25)), **kw})


EB = dict(proj=proj(), dy=p(0), proj2=None, dy2=None, dtype=MOE_BF16, perm=None, k=2, M=64, offsets=p(1), dx_in=None, dx=p(2))
SAVE = dict(gate=p(0), up=p(1), M=16, n=64, dtype=MOE_BF16, act=0, alpha=1.0, limit=7.0, rows=None, out=p(2), codes=p(3), scales=p(4))
REST = dict(codes=p(0), scales=p(1), numel=64, out=p(2), dtype=MOE_BF16)
AB = dict(codes=p(0), scales=p(1), dh=p(2), M=16, n=64, dtype=MOE_BF16, act=0, alpha=1.0, limit=7.0, w=p(3), perm=p(4), rows=None,
          dg=p(5), du=p(6), dw=p(7), h=p(8))
PB = dict(dX=p(0), inv=p(1), T=4, H=64, k=2, dx_in=None, dx=p(2), dtype=MOE_BF16)
NB = dict(r=p(0), w=p(1), dn=p(2), dr=p(3), eps=1e-6, T=4, H=64, dtype=MOE_BF16, din=p(4), dw=p(5), ws=p(6), ws_bytes=1 << 30)
INV, UNS, WS = MOE_ERR_INVALID, MOE_ERR_UNSUPPORTED, MOE_ERR_WORKSPACE


def call(fn, base, **kw):
    return getattr(_lib.load(), fn)(*{**base, **kw}.values(), None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(proj=None), INV, "NULL"), (dict(dy=None), INV, "NULL"), (dict(dx=None), INV, "NULL"), (dict(offsets=None), INV, "NULL"),
    (dict(proj2=other()), INV, "together"), (dict(dy2=p(5)), INV, "together"),
    (dict(proj2=other(bits=8), dy2=p(5)), INV, "formats"), (dict(proj2=other(n=64), dy2=p(5)), INV, "formats"),
    (dict(proj2=other(group_size=32), dy2=p(5)), INV, "formats"), (dict(proj2=other(weight=None), dy2=p(5)), INV, "non-NULL"),
    (dict(M=0), INV, "positive"), (dict(M=-5), INV, "positive"), (dict(M=(1 << 23) + 1), UNS, "above"),
    (dict(perm=p(3), k=0), INV, "top_k"), (dict(dtype=3), UNS, "pair"), (dict(dtype=MOE_F32), UNS, "pair"),
    (dict(proj=proj(sb_dtype=MOE_F32)), UNS, "pair"), (dict(proj=proj(bits=7)), INV, "bits"), (dict(proj=proj(k=100)), INV, "multiple"),
    (dict(proj=proj(n=100)), UNS, "multiple of 8"), (dict(proj=proj(n_experts=1025)), UNS, "1024"),
    (dict(proj=proj(n=1 << 21)), UNS, "2^20"), (dict(proj=proj(n=1 << 18, k=1 << 16)), UNS, "2^31"),
    (dict(dy=p(0, 8)), INV, "aligned"), (dict(dx=p(2, 4)), INV, "aligned"), (dict(dx_in=p(2, 8)), INV, "aligned"),
    (dict(proj2=other(), dy2=p(5, 2)), INV, "aligned"), (dict(proj=proj(weight=p(20, 8))), INV, "aligned"),
    (dict(dx=p(0)), INV, "overlaps"), (dict(dx=p(0, 64 * 128 * 2 - 16)), INV, "overlaps"), (dict(dx_in=p(2, 16)), INV, "overlaps"),
    (dict(proj2=other(), dy2=p(2, 32)), INV, "overlaps"), (dict(dx=p(20, 64)), INV, "experts"), (dict(dx=p(21)), INV, "experts"),
    (dict(proj=proj(n=8, k=1 << 20, sb_dtype=MOE_F32), dtype=MOE_F32, M=1 << 23, dy=p(0), dx=C.c_void_p(1 << 62)), UNS, "one launch"),
    (dict(proj2=other(), dy2=p(5), dx=p(25)), INV, "experts"), (dict(dx=p(1)), INV, "plan"), (dict(perm=p(2, 64)), INV, "plan"),
])
def test_expert_matmul_backward_refuses(kw, status, needle):
    assert call("moe_expert_matmul_backward", EB, **kw) == status
    assert needle in _lib.last_error()


KEPT = [
    (dict(codes=None), INV, "NULL"), (dict(scales=None), INV, "NULL"), (dict(M=0), INV, "positive"), (dict(n=0), INV, "positive"),
    (dict(n=48), UNS, "multiple of 32"), (dict(n=(1 << 20) + 32), UNS, "2^20"), (dict(M=(1 << 23) + 1), UNS, "above"),
    (dict(dtype=3), INV, "dtype"), (dict(act=4), INV, "kind"), (dict(codes=p(9, 8)), INV, "aligned"),
]


@pytest.mark.parametrize("kw,status,needle", KEPT + [
    (dict(gate=None), INV, "NULL"), (dict(up=None), INV, "NULL"), (dict(up=p(1, 8)), INV, "aligned"), (dict(out=p(2, 2)), INV, "aligned"),
    (dict(out=p(0, 16)), INV, "overlap"), (dict(codes=p(1)), INV, "overlap"), (dict(scales=p(3, 2047)), INV, "overlap"),
    (dict(scales=p(2, 2047)), INV, "overlap"),
])
def test_activation_save_refuses(kw, status, needle):
    assert call("moe_activation_save", SAVE, **kw) == status
    assert needle in _lib.last_error()


@pytest.mark.parametrize("kw,status,needle", [
    (dict(codes=None), INV, "NULL"), (dict(out=None), INV, "NULL"), (dict(numel=0), INV, "positive"), (dict(numel=48), UNS, "multiple"),
    (dict(numel=1 << 45), UNS, "2^44"), (dict(dtype=9), INV, "dtype"), (dict(out=p(2, 8)), INV, "aligned"), (dict(out=p(0)), INV, "overlaps"),
])
def test_checkpoint_restore_refuses(kw, status, needle):
    assert call("moe_checkpoint_restore", REST, **kw) == status
    assert needle in _lib.last_error()


@pytest.mark.parametrize("kw,status,needle", KEPT + [
    (dict(dh=None), INV, "NULL"), (dict(dg=None), INV, "NULL"), (dict(du=None), INV, "NULL"), (dict(act=3), INV, "no gate"),
    (dict(dh=p(2, 8)), INV, "aligned"), (dict(h=p(8, 8)), INV, "aligned"), (dict(du=p(5)), INV, "results overlap"),
    (dict(dw=p(6, 64)), INV, "results overlap"), (dict(h=p(2)), INV, "overlaps dh"), (dict(du=p(2, 16)), INV, "overlaps dh"),
    (dict(dg=p(0)), INV, "an input"), (dict(dw=p(3)), INV, "an input"), (dict(h=p(4)), INV, "an input"),
])
def test_activation_backward_refuses(kw, status, needle):
    assert call("moe_activation_backward", AB, **kw) == status
    assert needle in _lib.last_error()


@pytest.mark.parametrize("kw,status,needle", [
    (dict(dX=None), INV, "NULL"), (dict(inv=None), INV, "NULL"), (dict(dx=None), INV, "NULL"), (dict(T=0), INV, "positive"),
    (dict(H=-8), INV, "positive"), (dict(k=0), INV, "positive"), (dict(T=1 << 22, k=1 << 10), INV, "too large"),
    (dict(T=(1 << 23) + 1), UNS, "above"), (dict(H=60), UNS, "multiple of 8"), (dict(H=(1 << 20) + 8), UNS, "2^20"),
    (dict(dtype=5), INV, "dtype"), (dict(dX=p(0, 8)), INV, "aligned"), (dict(dx=p(0)), INV, "overlaps"), (dict(dx=p(1)), INV, "overlaps"),
    (dict(dx_in=p(2, 16)), INV, "overlaps"),
])
def test_permute_backward_refuses(kw, status, needle):
    assert call("moe_permute_backward", PB, **kw) == status
    assert needle in _lib.last_error()


@pytest.mark.parametrize("kw,status,needle", [
    (dict(r=None), INV, "NULL"), (dict(w=None), INV, "NULL"), (dict(dn=None), INV, "NULL"), (dict(din=None), INV, "NULL"),
    (dict(dw=None), INV, "NULL"), (dict(T=0), INV, "positive"), (dict(H=0), INV, "positive"), (dict(T=(1 << 23) + 1), UNS, "above"),
    (dict(H=60), UNS, "multiple of 8"), (dict(H=8200), UNS, "8192"), (dict(dtype=4), INV, "dtype"), (dict(eps=-1.0), INV, "eps"),
    (dict(eps=float("nan")), INV, "eps"), (dict(dn=p(2, 8)), INV, "aligned"), (dict(w=p(1, 2)), INV, "aligned"),
    (dict(din=p(0)), INV, "d_in overlaps"), (dict(din=p(2, 16)), INV, "d_in overlaps"), (dict(din=p(1)), INV, "d_in overlaps"),
    (dict(dw=p(4)), INV, "d_weight overlaps"), (dict(dw=p(2, 16)), INV, "d_weight overlaps"),
    (dict(T=100000, ws=None), WS, "workspace"), (dict(T=100000, ws_bytes=16), WS, "workspace"),
    (dict(T=100000, ws=p(6, 8)), WS, "aligned"),
])
def test_add_rmsnorm_backward_refuses(kw, status, needle):
    assert call("moe_add_rmsnorm_backward", NB, **kw) == status
    assert needle in _lib.last_error()


def test_add_rmsnorm_backward_workspace():
    size = _lib.load().moe_add_rmsnorm_backward_workspace_bytes
    assert size(1, 64) == 0
    assert 0 < size(8192, 2048) <= size(100000, 8192) <= 64 << 20
    for T, H in ((0, 64), (4, 60), (4, 8200), (4, 0), ((1 << 23) + 1, 64)):
        assert size(T, H) == 0
