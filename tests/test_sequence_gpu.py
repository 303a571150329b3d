"""Causal convolution, selective scan and the state-space head against the 64-bit recurrences of oracle/sequence.py.

Tolerances.  An output is a sum of products; in fp32 each factor is off by a few roundings u = 2^-24 and each passes at most T multiply-adds on its
way through the state (and back through the gradient's), so its error is at most (4 T + 32) u times the sum of the absolute terms.  The
terms have random signs, so that sum is some ten times the result's 2-norm: the 2-norm of the difference is held to 10 (4 T + 32) u of the
result's.  One rounding of a 16-bit output adds half a step, eps / 2."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

from freesound_classification_amd import functional as F  # noqa: E402
from freesound_classification_amd._lib import FscError  # noqa: E402
from freesound_classification_amd.networks.classifiers import SsmHead, TwoDimensionalCNNClassificationModel  # noqa: E402
from oracle import sequence as oseq  # noqa: E402

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def close(got, want, frames, what):
    got, want = got.detach().cpu().double(), want.detach().double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    return float((got - want).norm()), float(want.norm())


def check(got, want, frames, what):
    off, size = close(got, want, frames, what)
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    assert off <= (10 * (4 * frames + 32) * 2.0 ** -24 + half) * size + 1e-30, (what, off, size)


def make(shape, gen, dtype, scale=1.0):
    return (scale * torch.randn(shape, generator=gen)).to(dtype)


def on_device(t):
    return None if t is None else t.to(DEV)


def grads(outputs, leaves, cotangents):
    pairs = [(o, g) for o, g in zip(outputs, cotangents) if g is not None]
    return torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs], allow_unused=True)


def compare(fn, ofn, tensors, lengths, cotangents, frames, **kw):
    """Outputs and gradients of the operator and of the recurrence; tensors: name -> CPU tensor or None."""
    have = {k: v for k, v in tensors.items() if v is not None}
    dleaves = {k: v.to(DEV).requires_grad_() for k, v in have.items()}
    oleaves = {k: v.double().requires_grad_() for k, v in have.items()}
    dl = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = fn(dleaves, dl, **kw)
    want = ofn(oleaves, lengths, **kw)
    for name, g, w in zip(("y", "final"), got, want):
        check(g, w, frames, name)
    dg = grads(got, dleaves, [on_device(c) for c in cotangents])
    og = grads(want, oleaves, [None if c is None else c.double() for c in cotangents])
    for name, g, w in zip(have, dg, og):
        if w is not None:
            check(g, w, frames, "d" + name)
    return got, dict(zip(have, dg))


# ------------------------------------------------------------------------------------------------------------------ convolution
def conv_dev(p, lengths, silu=True):
    return F.causal_conv(p["x"], p["weight"], p.get("bias"), activation="silu" if silu else None, lengths=lengths, initial=p.get("initial"),
                         return_final=True)


def conv_ref(p, lengths, silu=True):
    return oseq.causal_conv(p["x"], p["weight"], p.get("bias"), silu, lengths, p.get("initial"))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n, t, d, k, opts", [
    (1, 1, 1, 1, ""), (2, 1, 8, 4, "bif"), (3, 2, 8, 4, "bilf"), (1, 3, 7, 8, "bilf"), (2, 65, 33, 3, "bil"), (2, 130, 64, 4, "b"),
    (4, 17, 260, 2, "f"), (2, 200, 12, 5, "bilfn"), (3, 64, 16, 6, "lfn"), (5, 9, 4, 7, "bi"), (1, 700, 3, 8, "bif"), (40, 5, 516, 4, "bil")])
def test_causal_conv(n, t, d, k, opts, dtype):
    """opts: b bias, i initial, l lengths (0, 1 and the whole among them), f a gradient of the final window, n no activation."""
    gen = torch.Generator().manual_seed(n + 10 * t + 100 * d + k)
    dt = DTYPES[dtype]
    p = dict(x=make((n, t, d), gen, dt), weight=make((d, k), gen, torch.float32, 0.5), bias=make((d,), gen, torch.float32) if "b" in opts else None,
             initial=make((n, k - 1, d), gen, dt) if "i" in opts else None)
    lengths = [(0, t, 1, t // 2, max(0, t - 1))[i % 5] for i in range(n)] if "l" in opts else None
    cot = [make((n, t, d), gen, dt), make((n, k - 1, d), gen, dt) if "f" in opts and k > 1 else None]
    compare(conv_dev, conv_ref, p, lengths, cot, 1, silu="n" not in opts)
    if cot[1] is not None and "i" in opts:
        compare(conv_dev, conv_ref, p, lengths, [None, cot[1]], 1, silu="n" not in opts)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n, d, k", [(1, 1, 1), (3, 7, 4), (48, 1536, 4), (2, 24, 8)])
def test_conv_frames_one_by_one(n, d, k, dtype):
    """A prompt, then single frames, equal the whole sequence, value for value: the same products in the same order."""
    gen = torch.Generator().manual_seed(d)
    dt = DTYPES[dtype]
    x, w, b = make((n, 11, d), gen, dt).to(DEV), make((d, k), gen, torch.float32).to(DEV), make((d,), gen, torch.float32).to(DEV)
    whole, last = F.causal_conv(x, w, b, return_final=True)
    y, window = F.causal_conv(x[:, :6], w, b, return_final=True)
    parts = [y]
    for i in range(6, 11):
        parts.append(F.causal_conv_step(x[:, i], window, w, b).unsqueeze(1))
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(window, last)
    again, more = F.causal_conv(x[:, 6:], w, b, initial=F.causal_conv(x[:, :6], w, b, return_final=True)[1], return_final=True)
    assert torch.equal(again, whole[:, 6:]) and torch.equal(more, last)


# ------------------------------------------------------------------------------------------------------------------------ scan
def scan_dev(p, lengths, softplus=True):
    return F.selective_scan(p["u"], p["dt"], p["a_log"], p["b"], p["c"], d=p.get("d"), z=p.get("z"), dt_bias=p.get("dt_bias"),
                            softplus=softplus, lengths=lengths, initial=p.get("initial"), return_final=True)


def scan_ref(p, lengths, softplus=True):
    return oseq.selective_scan(p["u"], p["dt"], p["a_log"], p["b"], p["c"], p.get("d"), p.get("z"), p.get("dt_bias"), softplus, lengths, p.get("initial"))


def scan_inputs(n, t, d, s, g, opts, dt, seed):
    gen = torch.Generator().manual_seed(seed)
    rate = torch.exp(torch.rand(d, generator=gen) * 4.6 - 6.9)
    raw = make((n, t, d), gen, torch.float32, 0.5)
    p = dict(u=make((n, t, d), gen, dt), dt=(raw if "p" not in opts else 0.1 * torch.rand((n, t, d), generator=gen)).to(dt),
             a_log=torch.log(torch.arange(1, s + 1).float()).repeat(d, 1) + make((d, s), gen, torch.float32, 0.2),
             b=make((n, t, g, s), gen, dt), c=make((n, t, g, s), gen, dt))
    if "d" in opts:
        p["d"] = make((d,), gen, torch.float32)
    if "z" in opts:
        p["z"] = make((n, t, d), gen, dt)
    if "b" in opts:
        p["dt_bias"] = rate + torch.log(-torch.expm1(-rate)) if "p" not in opts else 0.01 * torch.rand(d, generator=gen)
    if "i" in opts:
        p["initial"] = make((n, d, s), gen, torch.float32)
    lengths = [(t, 0, 1, t // 3, max(0, t - 1))[i % 5] for i in range(n)] if "l" in opts else None
    cot = [make((n, t, d), gen, dt), make((n, d, s), gen, torch.float32) if "f" in opts else None]
    return p, lengths, cot


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n, t, d, s, g, opts", [
    (1, 1, 1, 1, 1, ""), (2, 1, 64, 16, 1, "dzbif"), (2, 16, 64, 16, 1, "dzb"), (5, 17, 65, 16, 1, "dzbilf"), (3, 33, 70, 5, 2, "zbi"),
    (1, 50, 48, 64, 3, "dzb"), (2, 40, 130, 24, 1, "dbl"), (2, 5, 257, 8, 1, "dz"), (2, 30, 12, 3, 4, "dzbilfp"), (1, 31, 20, 33, 1, "bf"),
    (3, 48, 96, 2, 2, "ilp"), (70, 53, 256, 16, 1, "dzb"), (5, 20, 30, 17, 1, "dzblf")])
def test_selective_scan(n, t, d, s, g, opts, dtype):
    """opts: d skip, z gate, b time-step bias, i initial state, l lengths, f a gradient of the final state, p time steps as they are."""
    p, lengths, cot = scan_inputs(n, t, d, s, g, opts, DTYPES[dtype], n + t + d + s)
    compare(scan_dev, scan_ref, p, lengths, cot, t, softplus="p" not in opts)
    if cot[1] is not None:
        compare(scan_dev, scan_ref, p, lengths, [None, cot[1]], t, softplus="p" not in opts)


@pytest.mark.parametrize("n, t, d, s, g, opts", [(1, 400, 64, 16, 1, "dzbif"), (3, 333, 40, 20, 2, "dzbilf"), (2, 129, 16, 64, 1, "zb"), (1, 900, 5, 4, 1, "dzb")])
def test_selective_scan_in_segments(n, t, d, s, g, opts):
    """Few channels and many frames: time is cut into segments whose ends are joined."""
    p, lengths, cot = scan_inputs(n, t, d, s, g, opts, torch.float32, t)
    compare(scan_dev, scan_ref, p, lengths, cot, t)
    if cot[1] is not None:
        compare(scan_dev, scan_ref, p, lengths, [None, cot[1]], t)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n, d, s, g", [(1, 1, 1, 1), (3, 70, 16, 2), (2, 33, 5, 1), (4, 64, 64, 1), (2, 20, 30, 4)])
def test_scan_frames_one_by_one(n, d, s, g, dtype):
    """A prompt, then single frames: the recurrence, outputs and state, to the tolerance of the sequence."""
    p, _, _ = scan_inputs(n, 23, d, s, g, "dzbi", DTYPES[dtype], d)
    want, end = scan_ref({k: v.double() for k, v in p.items()}, None)
    q = {k: v.to(DEV) for k, v in p.items()}
    first = {k: v[:, :17] if v.dim() >= 3 and k != "initial" else v for k, v in q.items()}
    y, state = scan_dev(first, None)
    parts = [y]
    for i in range(17, 23):
        parts.append(F.selective_scan_step(q["u"][:, i], q["dt"][:, i], q["a_log"], q["b"][:, i], q["c"][:, i], state, d=q["d"], z=q["z"][:, i],
                                           dt_bias=q["dt_bias"]).unsqueeze(1))
    check(torch.cat(parts, 1), want, 23, "y")
    check(state, end, 23, "state")


# ---------------------------------------------------------------------------------------------------- what callers do to operators
def test_no_frames_and_no_sequences():
    w, a = torch.randn(8, 4, device=DEV), torch.zeros(8, 16, device=DEV)
    for n, t in ((2, 0), (0, 5)):
        x, rows = torch.randn(n, t, 8, device=DEV).requires_grad_(), torch.randn(n, t, 16, device=DEV)
        before, h0 = torch.randn(n, 3, 8, device=DEV).requires_grad_(), torch.randn(n, 8, 16, device=DEV).requires_grad_()
        wl, al = w.clone().requires_grad_(), a.clone().requires_grad_()
        y, final = F.causal_conv(x, wl, initial=before, return_final=True)
        assert y.shape == (n, t, 8) and torch.equal(final, before)
        gx, gw, gi = torch.autograd.grad([y, final], [x, wl, before], [torch.ones_like(y), torch.ones_like(final)])
        assert gx.shape == x.shape and not gw.any() and bool((gi == 1).all())
        y, final = F.selective_scan(x, x, al, rows, rows, initial=h0, return_final=True)
        assert y.shape == (n, t, 8) and torch.equal(final, h0)
        gx, ga, gi = torch.autograd.grad([y, final], [x, al, h0], [torch.ones_like(y), torch.ones_like(final)])
        assert gx.shape == x.shape and not ga.any() and bool((gi == 1).all())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_frames_that_do_not_exist_are_not_read(value):
    n, t, d, s = 4, 200, 36, 16
    p, _, (gy, _) = scan_inputs(n, t, d, s, 1, "dzbi", torch.float32, 5)
    lengths = torch.tensor([200, 0, 37, 112], dtype=torch.int32, device=DEV)
    there = torch.arange(t, device=DEV) < lengths[:, None]
    results = []
    for fill in (0.0, value):
        q = {k: v.to(DEV) for k, v in p.items()}
        for k in ("u", "dt", "b", "c", "z"):
            q[k] = torch.where(there.view((n, t) + (1,) * (q[k].dim() - 2)), q[k], torch.tensor(fill, device=DEV))
        g = torch.where(there[..., None], gy.to(DEV), torch.tensor(fill, device=DEV))
        leaves = {k: v.requires_grad_() for k, v in q.items()}
        out = list(scan_dev(leaves, lengths))
        out += torch.autograd.grad(out[0], list(leaves.values()), g)
        w = torch.full((d, 4), 0.3, device=DEV).requires_grad_()
        y, final = F.causal_conv(leaves["u"], w, lengths=lengths, return_final=True)
        out += [y, final] + list(torch.autograd.grad(y, [leaves["u"], w], g))
        results.append(out)
    for clean, filled in zip(*results):
        assert torch.equal(clean, filled) and torch.isfinite(filled).all()
    assert not results[1][0][~there].any()


def test_lengths_are_clamped():
    p, _, _ = scan_inputs(2, 20, 8, 16, 1, "dzb", torch.float32, 3)
    q = {k: v.to(DEV) for k, v in p.items()}
    odd, even = torch.tensor([-3, 1000], dtype=torch.int32, device=DEV), torch.tensor([0, 20], dtype=torch.int32, device=DEV)
    for a, b in zip(scan_dev(q, odd), scan_dev(q, even)):
        assert torch.equal(a, b)
    w = torch.randn(8, 4, device=DEV)
    for a, b in zip(*(F.causal_conv(q["u"], w, lengths=v, return_final=True) for v in (odd, even))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides_and_alignment(dtype):
    """Halves of a projection, odd offsets, transposed and expanded tensors: the same bits as contiguous copies."""
    n, t, d, s = 3, 37, 24, 16
    dt = DTYPES[dtype]
    gen = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device=DEV).to(dt)  # noqa: E731
    wide, rows = rnd(n, t, 3 * d + 1), rnd(n, t, 2 * s + 1)
    a_log, w = torch.rand(d, s, generator=gen, device=DEV), torch.rand(d, 4, generator=gen, device=DEV)
    z0 = rnd(n, d, t)
    views = dict(u=wide[..., 1:d + 1], dt=wide[..., d + 1:2 * d + 1], z=z0.transpose(1, 2), b=rows[..., 1:s + 1], c=rows[..., s + 1:])
    shared = rnd(1, t, s).expand(n, t, s)
    state = torch.zeros(n, d, s, device=DEV)
    results = []
    for copy in (lambda v: v, lambda v: v.contiguous().clone()):
        q = {k: copy(v).detach().requires_grad_() for k, v in views.items()}
        c = copy(shared).detach().requires_grad_()
        y = F.selective_scan(q["u"], q["dt"], a_log, q["b"], c, z=q["z"])
        out = [y] + list(torch.autograd.grad(y.float().sum(), [q[k] for k in ("u", "dt", "z", "b")] + [c]))
        y = F.causal_conv(q["u"], w)
        out += [y, F.causal_conv_step(q["u"][:, 3].detach(), copy(wide[:, :3, :d]).contiguous(), w)]
        out += list(torch.autograd.grad(y, [q["u"]], copy(wide[..., 2 * d:3 * d])))
        with torch.no_grad():
            out.append(F.selective_scan_step(q["u"][:, 5], q["dt"][:, 5], a_log, q["b"][:, 5], q["c"][:, 5], state.zero_(), z=q["z"][:, 5]))
        results.append([v.clone() for v in out])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_unaligned_states():
    n, d, s = 2, 9, 16
    gen = torch.Generator(device=DEV).manual_seed(2)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    u, b, a_log = rnd(n, d), rnd(n, s), rnd(d, s)
    base = rnd(n * d * s + 1)
    odd, even = base[1:].view(n, d, s), base[1:].clone().view(n, d, s)
    assert torch.equal(F.selective_scan_step(u, u, a_log, b, b, odd), F.selective_scan_step(u, u, a_log, b, b, even)) and torch.equal(odd, even)
    window = rnd(n * 3 * 8 + 1)
    x, w = rnd(n, 8), rnd(8, 4)
    odd, even = window[1:].view(n, 3, 8), window[1:].clone().view(n, 3, 8)
    first = float(window[0])
    assert torch.equal(F.causal_conv_step(x, odd, w), F.causal_conv_step(x, even, w)) and torch.equal(odd, even) and float(window[0]) == first


def test_offsets_beyond_32_bits():
    """Sequences 2^31 elements apart in one bf16 buffer."""
    t, d, s = 20, 64, 16
    far = 2 ** 31 + 64
    base = torch.empty(far + t * d, dtype=torch.bfloat16, device=DEV)
    u = base.as_strided((2, t, d), (far, d, 1))
    gen = torch.Generator(device=DEV).manual_seed(4)
    small = torch.randn(2, t, d, generator=gen, device=DEV).bfloat16()
    u.copy_(small)
    rows = torch.randn(2, t, s, generator=gen, device=DEV).bfloat16()
    a_log, w = torch.rand(d, s, device=DEV), torch.rand(d, 4, device=DEV)
    assert torch.equal(F.selective_scan(u, u, a_log, rows, rows, z=u), F.selective_scan(small, small, a_log, rows, rows, z=small))
    assert torch.equal(F.causal_conv(u, w), F.causal_conv(small, w))
    del base, u
    torch.cuda.empty_cache()


def test_short_sequences_in_long_padding():
    """One frame of 70 000 that exist, 2^15 elements apart: no offset from behind the end is formed in 32 bits."""
    t, d, far = 70000, 8, 2 ** 15
    base = torch.zeros(t * far + d, dtype=torch.bfloat16, device=DEV)
    x = base.as_strided((1, t, d), (0, far, 1))
    gen = torch.Generator(device=DEV).manual_seed(5)
    small = torch.randn(1, 1, d, generator=gen, device=DEV).bfloat16()
    x[:, :1] = small
    w, one = torch.rand(d, 4, generator=gen, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    results = []
    for v, lengths in ((x, one), (small, None)):
        leaf, wl = v.detach().requires_grad_(), w.clone().requires_grad_()
        y = F.causal_conv(leaf, wl, lengths=lengths)
        z = F.selective_scan(leaf, leaf, w, leaf[..., :4], leaf[..., 4:], lengths=lengths)
        g = torch.ones_like(small).expand(1, v.shape[1], d)
        results.append([y, z] + list(torch.autograd.grad([y, z], [leaf, wl], [g, g])))
    for a, b in zip(*results):
        assert torch.equal(a[:, :1] if a.dim() == 3 else a, b) and (a.dim() < 3 or not a[:, 1:].any())
    del base, x, results
    torch.cuda.empty_cache()


def test_frames_far_apart_are_copied():
    """A time stride above 2^26 elements, which the kernels refuse."""
    d, far = 4, 2 ** 26 + 4
    base = torch.zeros(2 * far, dtype=torch.bfloat16, device=DEV)
    x = base.as_strided((1, 2, d), (0, far, 1))
    x.copy_(torch.arange(2 * d, device=DEV).view(1, 2, d))
    w, rows = torch.ones(d, 2, device=DEV), torch.ones(1, 2, 3, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(F.causal_conv(x, w), F.causal_conv(x.contiguous(), w))
    assert torch.equal(F.selective_scan(x, x, w.new_zeros(d, 3), rows, rows), F.selective_scan(x.contiguous(), x.contiguous(), w.new_zeros(d, 3), rows, rows))


def test_one_frame_with_a_far_stride():
    """An axis of length 1 may have any stride."""
    gen = torch.Generator().manual_seed(5)
    x, w = make((2, 1, 8), gen, torch.float32).to(DEV), make((8, 4), gen, torch.float32).to(DEV)
    far = x.as_strided((2, 1, 8), (8, 2 ** 28, 1))
    assert torch.equal(F.causal_conv(far, w), F.causal_conv(x, w))


@pytest.mark.parametrize("n, t, s, lengths", [(2, 40, 16, [5, 33]), (2, 400, 5, [400, 77]), (1, 20, 64, None)])
def test_states_that_forget_everything(n, t, s, lengths):
    """exp(a_log) beyond fp32: such a state is delta u B of its frame alone, its rate's gradient 0, and padding behind the end changes nothing."""
    d = 12
    p, _, _ = scan_inputs(n, t, d, s, 1, "dzbi", torch.float32, 17)
    p["a_log"][::2, 0] = 100.0
    p["a_log"][1, :] = 90.0
    gen = torch.Generator().manual_seed(18)
    compare(scan_dev, scan_ref, p, lengths, [make((n, t, d), gen, torch.float32), make((n, d, s), gen, torch.float32)], t)


def test_steps_mark_what_they_change():
    """A graph that saved a state must notice that a step has moved it on."""
    gen = torch.Generator().manual_seed(6)
    x, w = make((2, 5, 8), gen, torch.float32).to(DEV), make((8, 4), gen, torch.float32).to(DEV)
    window = make((2, 3, 8), gen, torch.float32).to(DEV)
    y = F.causal_conv(x, w.requires_grad_(), initial=window)
    with torch.no_grad():
        F.causal_conv_step(x[:, 0], window, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    u, a = x, make((8, 4), gen, torch.float32).to(DEV)
    rows, state = make((2, 5, 4), gen, torch.float32).to(DEV), torch.zeros(2, 8, 4, device=DEV)
    y = F.selective_scan(u, u, a.requires_grad_(), rows, rows, initial=state)
    with torch.inference_mode():
        F.selective_scan_step(u[:, 0], u[:, 0], a, rows[:, 0], rows[:, 0], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_equal_inputs_give_equal_bits():
    p, lengths, cot = scan_inputs(6, 150, 200, 16, 2, "dzbil", torch.bfloat16, 9)
    dl = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    runs = []
    for _ in range(2):
        leaves = {k: v.to(DEV).requires_grad_() for k, v in p.items()}
        y, _ = scan_dev(leaves, dl)
        w = torch.full((200, 4), 0.25, device=DEV).requires_grad_()
        x = F.causal_conv(leaves["u"], w, lengths=dl)
        runs.append([y, x] + list(torch.autograd.grad([y, x], list(leaves.values()) + [w], [cot[0].to(DEV)] * 2)))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_gradients_against_differences():
    """The directional derivative of the 64-bit recurrence by central differences (step 1e-5: its own error is some 1e-9 of it) against the
    kernels' gradients in that direction."""
    p, _, (gy, gf) = scan_inputs(2, 40, 24, 16, 2, "dzbif", torch.float32, 21)
    leaves = {k: v.to(DEV).requires_grad_() for k, v in p.items()}
    got = torch.autograd.grad(scan_dev(leaves, None), list(leaves.values()), [gy.to(DEV), gf.to(DEV)])
    gen = torch.Generator().manual_seed(22)
    for name, g in zip(p, got):
        way = torch.randn(p[name].shape, generator=gen).double()

        def value(step):
            q = {k: v.double() + (step * way if k == name else 0.0) for k, v in p.items()}
            y, final = scan_ref(q, None)
            return float((y * gy.double()).sum() + (final * gf.double()).sum())

        want = (value(1e-5) - value(-1e-5)) / 2e-5
        have = float((g.cpu().double() * way).sum())
        scale = float(g.cpu().double().norm()) * float(way.norm())
        assert abs(have - want) <= 10 * (4 * 40 + 32) * 2.0 ** -24 * scale, name


def test_streams_and_graphs():
    """One call on a side stream; a forward and backward recorded into a graph and replayed with new inputs between eager calls; two calls at
    once on two streams."""
    n, t, d, s = 2, 300, 64, 16
    p, _, (gy, _) = scan_inputs(n, t, d, s, 1, "dzbi", torch.float32, 31)
    q = {k: v.to(DEV) for k, v in p.items()}
    w = torch.full((d, 4), 0.3, device=DEV)
    cot = gy.to(DEV)

    def both(v):
        leaves = {k: x.detach().requires_grad_() for k, x in v.items()}
        x = F.causal_conv(leaves["u"], w)
        y = F.selective_scan(x, leaves["dt"], leaves["a_log"], leaves["b"], leaves["c"], d=leaves["d"], z=leaves["z"], dt_bias=leaves["dt_bias"],
                             initial=leaves["initial"])
        return [y.detach()] + list(torch.autograd.grad(y, list(leaves.values()), cot))

    sets = [{k: v * f for k, v in q.items()} for f in (1.0, 0.7, 1.3)]
    want = [both(v) for v in sets]
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    for stream in (side, other):
        stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = both(sets[0])
    with torch.cuda.stream(other):
        second = both(sets[1])
    torch.cuda.synchronize()
    for got, ref in ((first, want[0]), (second, want[1])):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    static = {k: v.clone() for k, v in q.items()}
    state, window = torch.zeros(n, d, s, device=DEV), torch.zeros(n, 3, d, device=DEV)
    with torch.cuda.stream(side):
        both(static)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = both(static)
            with torch.no_grad():
                x1 = F.causal_conv_step(static["u"][:, 0], window, w)
                y1 = F.selective_scan_step(x1, static["dt"][:, 0], static["a_log"], static["b"][:, 0], static["c"][:, 0], state)
        for turn in (1, 2, 0, 1):
            for k, v in sets[turn].items():
                static[k].copy_(v)
            h, f = state.clone(), window.clone()
            graph.replay()
            eager = both(sets[turn])
            x2 = F.causal_conv_step(static["u"][:, 0], f, w)
            y2 = F.selective_scan_step(x2, static["dt"][:, 0], static["a_log"], static["b"][:, 0], static["c"][:, 0], h)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(kept, want[turn])) and all(torch.equal(a, b) for a, b in zip(eager, want[turn]))
            assert torch.equal(y1, y2) and torch.equal(h, state) and torch.equal(f, window)


def test_refusals():
    x, w, a = torch.randn(2, 5, 8, device=DEV), torch.randn(8, 4, device=DEV), torch.zeros(8, 16, device=DEV)
    rows = torch.randn(2, 5, 16, device=DEV)
    l32 = torch.tensor([5, 3], dtype=torch.int32, device=DEV)
    state, window = torch.zeros(2, 8, 16, device=DEV), torch.zeros(2, 3, 8, device=DEV)
    bad = [
        lambda: F.causal_conv(x.double(), w), lambda: F.causal_conv(x, w.half()), lambda: F.causal_conv(x, w[:7]),
        lambda: F.causal_conv(x, torch.zeros(8, 9, device=DEV)), lambda: F.causal_conv(x, w, bias=torch.zeros(7, device=DEV)),
        lambda: F.causal_conv(x, w, lengths=l32.long()), lambda: F.causal_conv(x, w, lengths=l32[:1]), lambda: F.causal_conv(x, w, lengths=l32.cpu()),
        lambda: F.causal_conv(x, w, initial=window[:, :2]), lambda: F.causal_conv(x, w, initial=window.bfloat16()),
        lambda: F.causal_conv_step(x[:, 0], window.transpose(0, 1), w), lambda: F.causal_conv_step(x[:, 0].bfloat16(), window, w),
        lambda: F.causal_conv_step(x[:, 0].requires_grad_(), window, w), lambda: F.causal_conv_step(x[:, 0], window.clone().requires_grad_(), w),
        lambda: F.selective_scan(x, x.bfloat16(), a, rows, rows), lambda: F.selective_scan(x, x, a, rows[..., :8], rows),
        lambda: F.selective_scan(x, x, a, rows.view(2, 5, 1, 16).expand(2, 5, 3, 16), rows), lambda: F.selective_scan(x, x, a, rows, rows.cpu()),
        lambda: F.selective_scan(x, x, torch.zeros(8, 65, device=DEV), rows, rows), lambda: F.selective_scan(x, x, a.half(), rows, rows),
        lambda: F.selective_scan(x, x, a, rows, rows.view(2, 5, 1, 16).expand(2, 5, 2, 16)), lambda: F.selective_scan(x, x, a, rows, rows, initial=state[:1]),
        lambda: F.selective_scan(x, x, a, rows, rows, z=x[:, :4]), lambda: F.selective_scan(x, x, a, rows, rows, d=torch.zeros(8, 1, device=DEV)),
        lambda: F.selective_scan_step(x[:, 0], x[:, 0], a, rows[:, 0], rows[:, 0], state.half()),
        lambda: F.selective_scan_step(x[:, 0], x[:, 0], a, rows[:, 0], rows[:, 0], state.transpose(1, 2)),
        lambda: F.selective_scan_step(x[:, 0], x[:, 0], a.clone().requires_grad_(), rows[:, 0], rows[:, 0], state),
    ]
    for i, fn in enumerate(bad):
        with pytest.raises(FscError):
            fn()
            pytest.fail("call %d was not refused" % i)
    with pytest.raises(RuntimeError):                               # no second derivatives
        leaf = x.detach().clone().requires_grad_()
        (g,) = torch.autograd.grad(F.causal_conv(leaf, w).sum(), [leaf], create_graph=True)
        g.sum().backward()


# ------------------------------------------------------------------------------------------------------------------------ head
class NS(dict):
    __getattr__ = dict.__getitem__


@pytest.mark.parametrize("shape", [(3, 12, 8, 23), (2, 37, 1, 90), (4, 20, 2, 1)])
def test_ssm_head(shape):
    torch.manual_seed(sum(shape))
    head = SsmHead(shape[1])
    with torch.no_grad():
        head.norm.weight.uniform_(0.5, 1.5)
        head.norm.bias.normal_(0, 0.2)
        head.conv_bias.normal_(0, 0.2)
    x = torch.randn(shape)
    gy = torch.randn(shape[0], head.inner)
    p = {k: v.detach().double().requires_grad_() for k, v in head.named_parameters()}
    ox = x.double().requires_grad_()
    want = oseq.ssm_head(ox, p, head.inner, head.rank, head.states)
    og = torch.autograd.grad(want, [ox] + list(p.values()), gy.double())
    head = head.to(DEV)
    dx = x.to(DEV).requires_grad_()
    got = F.ssm_head(dx, head)
    dg = torch.autograd.grad(got, [dx] + list(head.parameters()), gy.to(DEV))
    # (projections of up to 512 terms and two norms around the operators: 512 roundings more)
    for name, g, w in zip(["y", "x"] + list(p), [got] + list(dg), [want] + list(og)):
        check(g, w, shape[3] + 128, name)


def experiment(optimizer, features="mel_1024_512_64", base=8):
    return NS(config=NS(
        network=NS(num_conv_blocks=3, start_deep_supervision_on=1, conv_base_depth=base, growth_rate=1.5, output_dropout=0.0, aggregation_type="ssm"),
        data=NS(features=features, _input_dim=64, _n_classes=80),
        train=NS(accumulation_steps=1, optimizer=optimizer, learning_rate=1e-3, weight_decay=0.01, scheduler="1cycle_0.0001_0.001")))


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_model_trains_eagerly_and_replayed(optimizer):
    """The tagger with state-space heads under AdamW: parameters of every head get gradients, a recorded step replays like eager ones."""
    from freesound_classification_amd.ops.training import CapturedTrainingStep, make_step
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        torch.manual_seed(11)
        model = TwoDimensionalCNNClassificationModel(experiment(optimizer), device=DEV)
        assert len(model.ssms) == 2 and model.output_transform[1].in_features == 512
        model.train()
        model.make_optimizer(max_steps=12)
        gen = torch.Generator(device=DEV).manual_seed(3)
        x = 0.1 * torch.randn(8, 22050, 1, device=DEV, generator=gen)
        y = (torch.rand(8, 80, device=DEV, generator=gen) < 0.05).float()
        make_step(model.scheduler, step=1)
        model.training_step(x, y, step_optimizer=False)
        for k, p in model.ssms.named_parameters():
            assert p.grad is not None and torch.isfinite(p.grad).all() and bool(p.grad.any()), k
        model.optimizer.step()
        model.optimizer.zero_grad()
        state = {k: v.clone() for k, v in model.state_dict().items()}
        import copy
        moments = copy.deepcopy(model.optimizer.state_dict())

        def run(step):
            model.scheduler.epoch = 0
            logits = []
            for i in range(3):
                make_step(model.scheduler, step=2 + i)
                logits.append(step(x, y)[0].detach().clone())
                torch.cuda.synchronize()
            return logits

        eager = run(model.training_step)
        model.load_state_dict(state)
        model.optimizer.load_state_dict(copy.deepcopy(moments))
        step = CapturedTrainingStep(model, x, y)
        replayed = run(step)
        # step 0 runs on equal weights (atomics in split products and norms: 1e-4); an update moves a weight by at most some lr = 1e-3
        for i, (a, b) in enumerate(zip(eager, replayed)):
            assert float((a - b).abs().max()) <= (1e-4 if i == 0 else 2e-2) * max(1.0, float(a.abs().max())), i
        assert all(int(s["step"]) == 4 for s in model.optimizer.state.values())
        model.eval()
        with torch.no_grad():
            assert torch.isfinite(model(x)["class_logits"]).all()
        model.close()
    torch.cuda.synchronize()


def test_training_command(tmp_path):
    import train_2d_cnn as drv
    argv = ("--synthetic 48 --synthetic_test 4 --epochs 1 --batch_size 8 --n_folds 2 --folds 0 --num_conv_blocks 2 --conv_base_depth 8 "
            "--growth_rate 1.5 --start_deep_supervision_on 1 --features mel_1024_512_64 --scheduler 1cycle_0.0001_0.001 --lr 0.001 "
            "--optimizer adamw8 --weight_decay 0.01 --num_workers 0 --aggregation_type ssm --experiments_dir %s" % tmp_path).split()
    _, scores = drv.main(argv=argv)
    assert len(scores[0]) == 1 and np.isfinite(scores[0][0])
