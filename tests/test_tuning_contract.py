"""What the tuning entry points promise about the tensors they are given and the memory they ask for, checked on the host
before any launch."""
import pytest

torch = pytest.importorskip("torch")

from ffai_amd import tuning  # noqa: E402


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
