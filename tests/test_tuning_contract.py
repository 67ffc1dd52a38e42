"""What the tuning entry points promise about the tensors they are given and the memory they ask for, checked on the host
before any launch."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from ffai_amd import _lib, tuning  # noqa: E402
from ffai_amd._lib import MOE_BF16, MOE_F32, Lora  # noqa: E402
from ffai_amd.layer import MoERouter  # noqa: E402


# -------------------------------------------------------- adapters' memory --

def adapters():
    """Two adapters whose scale is the front of a longer tensor."""
    scale = torch.ones(8)
    l = tuning.LoRAAdapters(torch.zeros(2, 8, 16), torch.zeros(2, 24, 8), scale[:2])
    return l, scale, torch.zeros(3, 16), torch.zeros(3, dtype=torch.int32)


@pytest.mark.parametrize("change,needle", [
    (lambda wide: wide[:1], r"scale must be \[2\], got \[1\]"),
    (lambda wide: wide[:4], r"scale must be \[2\], got \[4\]"),
    (lambda wide: wide[::4], "scale must be contiguous"),
    (lambda wide: wide[:2].view(torch.int32), "scale dtype"),
    (lambda wide: wide[:2].view(1, 2), r"scale must be \[2\], got \[1, 2\]"),
])
def test_scale_checked_each_call(change, needle):
    """A scale whose memory is set to a view of another length, type or spacing is refused, also at the same address."""
    l, wide, x, ad = adapters()
    at = l.scale.data_ptr()
    l.scale.data = change(wide)
    assert l.scale.data_ptr() == at
    for call in (lambda: l.apply(x, ad), lambda: l.backward(x, torch.zeros(3, 24), ad)):
        with pytest.raises(ValueError, match=needle):
            call()


def test_scale_of_the_same_kind_is_taken():
    l, wide, x, ad = adapters()
    l.scale.data = wide[4:6]
    with pytest.raises(ValueError, match="on a GPU"):  # past the adapters' own checks
        l.apply(x, ad)
    assert l._current().scale == wide.data_ptr() + 16


# -------------------------------------------------------------- workspaces --

def backward_bytes(T, G, K, N, R, dt=MOE_BF16):
    l = Lora(1 << 45, 1 << 46, None, dt, R, N, K, G)
    return _lib.load().moe_lora_backward_workspace_bytes(C.byref(l), T)


@pytest.mark.parametrize("T,G,K,N,R", [
    (512, 512, 4096, 4096, 64), (64, 64, 4096, 4096, 64), (2048, 512, 4096, 4096, 64), (4096, 1024, 8192, 8192, 128),
    (1, 1024, 2048, 768, 16), (4096, 8, 2048, 2048, 16), (333, 1, 1024, 384, 8), (40000, 1024, 2048, 768, 16),
])
@pytest.mark.parametrize("dt", [MOE_BF16, MOE_F32])
def test_backward_workspace_follows_the_rows(T, G, K, N, R, dt):
    """Partial gradients are kept for chunks of at least 64 rows, and for one shorter chunk of each adapter that has such
    a one: no memory for adapters that have few rows or none."""
    part = 4 * R * (K + N)
    rows = T * (8 * R + 8) + 4 * 1024 * (T // 1024 + 1) + 12 * (G + 1)  # inner sums, the plan's lists and its chunks
    assert backward_bytes(T, G, K, N, R, dt) <= 2 * (T // 64) * part + rows + 10 * 256
    # and it is what more rows need, at most
    sizes = [backward_bytes(t, G, K, N, R, dt) for t in [*range(1, 300), 511, 512, 513, 1000, T + 300, T + 301, 2 * T + 300]]
    assert sizes[:-3] == sorted(sizes[:-3]) and sizes[-3:] == sorted(sizes[-3:])


# ---------------------------------------------------------------- autograd --

def leaf(*shape):
    return torch.zeros(*shape).requires_grad_(True)


def refused_calls():
    """(call, the tensor it names) with a tensor that requires a gradient where autograd would have to record the call, or
    to know of a write."""
    r = MoERouter(8, 2)
    x, ad, y, dy = torch.zeros(3, 16), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 24), torch.zeros(3, 24)
    lg, idx = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    a, b = torch.zeros(2, 8, 16), torch.zeros(2, 24, 8)
    l = tuning.LoRAAdapters(a, b, torch.ones(2))
    g, Y, inv, w = torch.zeros(3, 8), torch.zeros(6, 8), torch.zeros(6, dtype=torch.int32), torch.zeros(3, 2)
    return [
        (lambda: tuning.balance_loss(r, leaf(4, 8), idx), "logits"),
        (lambda: tuning.router_backward(r, lg, idx, out=leaf(4, 8)), "out"),
        (lambda: tuning.unpermute_backward(g, Y, inv, w, dY=leaf(6, 8)), "dY"),
        (lambda: l.apply(leaf(3, 16), ad, y), "x"),
        (lambda: l.apply(x, ad, leaf(3, 24)), "y"),
        (lambda: l.apply(x, ad, y, out=leaf(3, 24)), "out"),
        (lambda: tuning.LoRAAdapters(leaf(2, 8, 16), b).apply(x, ad, y), "a"),
        (lambda: tuning.LoRAAdapters(a, leaf(2, 24, 8)).apply(x, ad, y), "b"),
        (lambda: tuning.LoRAAdapters(a, b, leaf(2)).apply(x, ad, y), "scale"),
        (lambda: l.backward(x, dy, ad, dx=leaf(3, 16)), "dx"),
        (lambda: l.backward(x, dy, ad, dx=x, dx_out=leaf(3, 16)), "dx_out"),
    ]


@pytest.mark.parametrize("i", range(11))
def test_tensors_that_require_a_gradient_are_refused_while_autograd_records(i):
    call, name = refused_calls()[i]
    with pytest.raises(ValueError, match=f"{name} requires a gradient"):
        call()
    for quiet in (torch.no_grad(), torch.inference_mode()):
        with quiet, pytest.raises(ValueError, match="on a GPU"):  # past that check
            call()


def test_gradient_calls_read_tensors_that_require_one():
    """What gradients are computed from may require one itself: the results are plain."""
    r, idx = MoERouter(8, 2), torch.zeros(4, 2, dtype=torch.int32)
    l = tuning.LoRAAdapters(leaf(2, 8, 16), leaf(2, 24, 8))
    ad, inv = torch.zeros(3, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    for call in (lambda: tuning.router_backward(r, leaf(4, 8), idx, leaf(4, 2)), lambda: l.backward(leaf(3, 16), leaf(3, 24), ad),
                 lambda: tuning.unpermute_backward(leaf(3, 8), leaf(6, 8), inv, leaf(3, 2))):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
