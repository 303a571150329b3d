"""Sequence operators on the device, at the edges of what is allowed: empty axes, values that are not finite, forward derivatives, states from elsewhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

from freesound_classification_amd import functional as F  # noqa: E402

DEV = "cuda:0"


def dirty(*shapes):
    """Blocks of NaN of these sizes go back to the allocator: what is not written afterwards is seen."""
    blocks = [torch.full(shape, float("nan"), device=DEV) for shape in shapes for _ in range(8)]
    torch.cuda.synchronize()
    del blocks


@pytest.mark.parametrize("n, t, d", [(0, 300, 8), (2, 300, 0), (2, 5, 0), (0, 300, 0), (2, 0, 0)])
def test_empty_axes(n, t, d):
    """No sequences or no channels, at lengths where time would be cut: empty outputs, and gradients of what is not empty are zeros."""
    x = torch.zeros(n, t, d, device=DEV).requires_grad_()
    w, bias = torch.ones(d, 4, device=DEV).requires_grad_(), torch.ones(d, device=DEV).requires_grad_()
    y, final = F.causal_conv(x, w, bias, return_final=True)
    assert y.shape == (n, t, d) and final.shape == (n, 3, d)
    for leaf, g in zip((x, w, bias), torch.autograd.grad([y, final], [x, w, bias], [torch.ones_like(y), torch.ones_like(final)])):
        assert g.shape == leaf.shape and not g.any()
    a, skip = torch.zeros(d, 16, device=DEV).requires_grad_(), torch.ones(d, device=DEV).requires_grad_()
    b, c = (torch.ones(n, t, 16, device=DEV).requires_grad_() for _ in range(2))
    y, final = F.selective_scan(x, x, a, b, c, d=skip, z=x, return_final=True)
    assert y.shape == (n, t, d) and final.shape == (n, d, 16)
    leaves = (x, a, b, c, skip)
    dirty((n, t, 16), (n, t, 16))
    for leaf, g in zip(leaves, torch.autograd.grad([y, final], leaves, [torch.ones_like(y), torch.ones_like(final)])):
        assert g.shape == leaf.shape and not g.any() and bool(torch.isfinite(g).all())
