"""Refusals of the gradient calls where buffers meet that their contract keeps apart."""
import pytest

from test_expert_grad_abi import INV, NB, call, p

from ffai_amd import _lib

ROWS = 100000 * 64 * 2  # bytes of the rows below


@pytest.mark.parametrize("kw,needle", [
    (dict(ws=p(0)), "rows"), (dict(ws=p(0, ROWS - 16)), "rows"), (dict(ws=p(2, 64)), "rows"), (dict(ws=p(3, 1 << 20)), "rows"),
    (dict(ws=p(4)), "rows"), (dict(ws=p(2), din=p(2)), "rows"), (dict(r=p(6, 4096)), "rows"), (dict(ws=p(1)), "weight"),
    (dict(w=p(6, 128)), "weight"), (dict(ws=p(5)), "weight"), (dict(dw=p(6, 16)), "weight"),
])
def test_add_rmsnorm_backward_keeps_its_workspace(kw, needle):
    """The first launch writes the blocks' shares there while other blocks still read the rows."""
    assert call("moe_add_rmsnorm_backward", NB, **{**dict(T=100000), **kw}) == INV
    assert "workspace" in _lib.last_error() and needle in _lib.last_error()
