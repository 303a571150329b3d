"""Sequence operators on the device, at the edges of what is allowed: empty axes, values that are not finite, forward derivatives, states from elsewhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

from freesound_classification_amd import functional as F  # noqa: E402
from oracle import sequence as oseq  # noqa: E402

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


def same_kinds(got, want, frames, what):
    """Infinities and NaN where the definition has them, of the same sign; the others to 10 (4 T + 32) u of their 2-norm, as in the sequence tests."""
    got, want = got.detach().cpu().double(), want.detach()
    assert got.shape == want.shape, what
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want)), (what, kind.__name__, int((kind(got) != kind(want)).sum()))
    fine = torch.isfinite(want)
    off = float((got[fine] - want[fine]).norm())
    assert off <= 10 * (4 * frames + 32) * 2.0 ** -24 * float(want[fine].norm()) + 1e-30, (what, off)


@pytest.mark.parametrize("where", ["u", "dt", "b", "c"])
@pytest.mark.parametrize("n, t, d, s, g, at, length", [
    (1, 40, 64, 16, 1, 9, None), (1, 40, 70, 5, 1, 9, None), (2, 40, 70, 16, 2, 20, None), (1, 21, 12, 3, 1, 0, None), (1, 30, 33, 24, 1, 17, None),
    (1, 20, 20, 33, 1, 3, None), (1, 20, 5, 1, 1, 3, None), (1, 400, 40, 5, 1, 333, None), (1, 400, 70, 17, 2, 20, None), (2, 40, 70, 5, 1, 32, 33),
    (2, 40, 64, 16, 1, 20, 21), (1, 300, 24, 12, 1, 199, 200)])
def test_infinities_stay_infinities(n, t, d, s, g, at, length, where):
    """One infinite value in the last channel (the last state of the last group) at frame `at`, everything else positive, so that no infinities of two signs meet: outputs and
    gradients are infinite where the recurrence's are, whatever states and channels the lanes are padded with, and the frames behind a
    sequence's end get their zeros."""
    gen = torch.Generator().manual_seed(d + s + at)
    pos = lambda *shape: 0.2 + torch.rand(*shape, generator=gen)  # noqa: E731
    p = dict(u=pos(n, t, d), dt=pos(n, t, d) - 1.0, a_log=pos(d, s), b=pos(n, t, g, s), c=pos(n, t, g, s), d=pos(d), z=pos(n, t, d), dt_bias=pos(d) - 1.0,
             initial=pos(n, d, s))
    p[where][0, at].view(-1)[-1] = float("inf")
    lengths = None if length is None else [length] + [t] * (n - 1)
    cot = pos(n, t, d), pos(n, d, s)
    if length is not None:
        cot[0][0, length:] = float("nan")                    # (never read)
    dev = {k: v.to(DEV).requires_grad_() for k, v in p.items()}
    ref = {k: v.double().requires_grad_() for k, v in p.items()}
    got = F.selective_scan(dev["u"], dev["dt"], dev["a_log"], dev["b"], dev["c"], d=dev["d"], z=dev["z"], dt_bias=dev["dt_bias"], initial=dev["initial"],
                           lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV), return_final=True)
    want = oseq.selective_scan(ref["u"], ref["dt"], ref["a_log"], ref["b"], ref["c"], ref["d"], ref["z"], ref["dt_bias"], True, lengths, ref["initial"])
    for name, a, b in zip(("y", "final"), got, want):
        same_kinds(a, b, t, name)
    grads = torch.autograd.grad(got, list(dev.values()), [v.to(DEV) for v in cot])
    clean = [torch.nan_to_num(v.double(), nan=0.0) for v in cot]
    for name, a, b in zip(p, grads, torch.autograd.grad(want, list(ref.values()), clean)):
        same_kinds(a, b, t, "d" + name)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("n, t, d, k, at, length, initial", [
    (1, 24, 8, 4, 23, None, True), (1, 24, 8, 4, 8, None, False), (2, 100, 12, 8, 62, 64, True), (1, 70, 5, 3, 69, None, False), (1, 9, 8, 2, 0, 1, True),
    (2, 40, 64, 4, 7, None, True), (1, 33, 7, 5, 30, 32, False), (1, 3000, 8, 4, 1500, None, True)])
def test_what_is_not_finite_stays_with_its_taps(n, t, d, k, at, length, initial, value):
    """One value of x that is not finite, no activation: each tap's gradient holds it where the tap meets it in a frame that exists, the last taps of a
    sequence's last frames do not; the strips that time is cut into and the frames behind the end do not spread it."""
    gen = torch.Generator().manual_seed(t + k)
    pos = lambda *shape: 0.2 + torch.rand(*shape, generator=gen)  # noqa: E731
    p = dict(x=pos(n, t, d), weight=pos(d, k), bias=pos(d))
    if initial:
        p["initial"] = pos(n, k - 1, d)
    p["x"][0, at, d - 1] = value
    lengths = None if length is None else [length] + [t] * (n - 1)
    cot = pos(n, t, d), pos(n, k - 1, d)
    dev = {key: v.to(DEV).requires_grad_() for key, v in p.items()}
    ref = {key: v.double().requires_grad_() for key, v in p.items()}
    got = F.causal_conv(dev["x"], dev["weight"], dev["bias"], activation=None, initial=dev.get("initial"),
                        lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV), return_final=True)
    want = oseq.causal_conv(ref["x"], ref["weight"], ref["bias"], False, lengths, ref.get("initial"))
    for name, a, b in zip(("y", "final"), got, want):
        same_kinds(a, b, 1, name)
    grads = torch.autograd.grad(got, list(dev.values()), [v.to(DEV) for v in cot])
    for name, a, b in zip(p, grads, torch.autograd.grad(want, list(ref.values()), [v.double() for v in cot])):
        same_kinds(a, b, 1 if name != "weight" and name != "bias" else n * t, "d" + name)
