"""Refusals of the gradient calls where buffers meet that their contract keeps apart."""
import pytest

from test_expert_grad_abi import AB, INV, NB, SAVE, call, p

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


@pytest.mark.parametrize("kw", [dict(rows=p(2)), dict(rows=p(3, 2044)), dict(rows=p(4, 60)), dict(out=p(9, 4080), rows=p(9, 4096))])
def test_activation_save_keeps_the_row_count(kw):
    """Every block reads it, and some write before others start."""
    assert call("moe_activation_save", SAVE, **kw) == INV
    assert "n_rows" in _lib.last_error() or "overlap" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(rows=p(5)), dict(rows=p(6, 2044)), dict(rows=p(7, 60)), dict(rows=p(8, 1024)),
                                dict(dg=p(2), rows=p(2, 4))])
def test_activation_backward_keeps_the_row_count(kw):
    assert call("moe_activation_backward", AB, **kw) == INV
    assert "input" in _lib.last_error()
