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


def test_single_frames_take_the_rates_of_the_sequence():
    """exp(a_log) of large a_log beside small time steps.  h' = exp(-r) h, r = dt exp(a_log) <= 3, in units u = 2^-24: exp(a_log) is off by 2 (one
    unit in the last place), dt log2(e) by 2 (the constant and the product), their product by 1, each times r in the result; exp2 by 2 and the
    last product by 1: (5 r + 3) u.  (An exponential by way of a rounded a_log log2(e) is off by a_log u, here up to 80, times r.)"""
    n, d = 64, 48
    gen = torch.Generator().manual_seed(41)
    a_log = 40 + 40 * torch.rand(d, 1, generator=gen)
    r = 0.1 + 2.9 * torch.rand(n, d, generator=gen).double()
    dt = (r / torch.exp(a_log.double())[:, 0]).float()
    h = torch.randn(n, d, 1, generator=gen)
    r = dt.double() * torch.exp(a_log.double())[:, 0]
    want = torch.exp(-r) * h[..., 0].double()
    zeros, rows = torch.zeros(n, d, device=DEV), torch.zeros(n, 1, device=DEV)
    state = h.to(DEV)
    F.selective_scan_step(zeros, dt.to(DEV), a_log.to(DEV), rows, rows, state, softplus=False)
    _, final = F.selective_scan(zeros[:, None], dt.to(DEV)[:, None], a_log.to(DEV), rows[:, None], rows[:, None], softplus=False, initial=h.to(DEV),
                                return_final=True)
    for got in (state, final):
        assert bool(((got[..., 0].cpu().double() - want).abs() <= (5 * r + 3) * 2.0 ** -24 * want.abs()).all())
