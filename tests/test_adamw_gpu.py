"""AdamW over many tensors: 32-bit moments against the formulas in 64 bits, 8-bit moments against the formulas in fp32 operation by operation
(oracle/sequence.py), where the held patterns are equal bit for bit."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

from freesound_classification_amd._lib import FscError  # noqa: E402
from freesound_classification_amd.ops.training import FusedAdamW  # noqa: E402
from oracle import sequence as oseq  # noqa: E402

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = [1, 3, 255, 256, 257, 1000, 4095, 4096, 4097, 70001]


def parameters(sizes, dtype, gen, offset=0):
    """Leaves in one buffer each `offset` elements off the start of their storage."""
    out = []
    for count in sizes:
        base = (0.05 * torch.randn(count + offset, generator=gen)).to(dtype).to(DEV)
        out.append(torch.nn.Parameter(base[offset:]))
    return out


def gradients(params, gen, offset=0):
    for p in params:
        size = torch.exp(2 * torch.randn(p.numel() + offset, generator=gen)) * 1e-3
        p.grad = (size * torch.randn(p.numel() + offset, generator=gen)).to(p.dtype).to(DEV)[offset:]


def host(t):
    return t.detach().cpu().float().numpy()


HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def _hyper():
    return dict(lr=HYPER["lr"], beta1=HYPER["betas"][0], beta2=HYPER["betas"][1], eps=HYPER["eps"], weight_decay=HYPER["weight_decay"])


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_32_bit_moments(dtype, offset):
    """Five roundings an update at most of u = 2^-24 in each moment and step, and one of the parameter's type: 8 (steps + 1) u of its size."""
    gen = torch.Generator().manual_seed(1)
    params = parameters(SIZES, DTYPES[dtype], gen, offset)
    opt = FusedAdamW(params, **HYPER)
    m, v = [np.zeros(c) for c in SIZES], [np.zeros(c) for c in SIZES]
    for step in (1, 2, 3):
        gradients(params, gen, offset)
        before = [host(p).astype(np.float64) for p in params]
        opt.step()
        for i, p in enumerate(params):
            q, m[i], v[i] = oseq.adamw(before[i], host(p.grad).astype(np.float64), m[i], v[i], step, **_hyper())
            half = 0.0 if dtype == "fp32" else torch.finfo(p.dtype).eps / 2
            small = 0.0 if dtype == "fp32" else float(torch.finfo(p.dtype).smallest_normal) * torch.finfo(p.dtype).eps      # (fp16 below its normal numbers)
            u = 8 * (step + 1) * 2.0 ** -24
            assert np.all(np.abs(host(p) - q) <= (half + u) * np.abs(q) + u * (HYPER["lr"] * 32 + np.abs(before[i])) + small), (step, i)
            assert np.all(np.abs(host(opt.state[p]["exp_avg"]) - m[i]) <= u * (np.abs(m[i]) + np.abs(host(p.grad)) + np.abs(m[i]).max())), (step, i)
            assert np.all(np.abs(host(opt.state[p]["exp_avg_sq"]) - v[i]) <= u * np.abs(v[i]) + 1e-37), (step, i)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_8_bit_moments_bit_for_bit(dtype, offset):
    gen = torch.Generator().manual_seed(2)
    params = parameters(SIZES, DTYPES[dtype], gen, offset)
    opt = FusedAdamW(params, state_bits=8, seed=77, **HYPER)
    held = [[np.zeros(c, np.uint8)] * 2 for c in SIZES]
    scales = [[np.zeros(-(-c // 256), np.float32)] * 2 for c in SIZES]
    for step in (1, 2, 3, 4):
        gradients(params, gen, offset)
        before = [host(p) for p in params]
        opt.step()
        for i, p in enumerate(params):
            q, held[i], scales[i] = oseq.adamw8(before[i], host(p.grad), held[i], scales[i], 77 + i, step, **_hyper())
            assert np.array_equal(host(p), host(torch.from_numpy(q).to(p.dtype))), (step, i)
            st = opt.state[p]
            for j, key in enumerate(("exp_avg", "exp_avg_sq_root")):
                assert np.array_equal(st[key].view(torch.uint8).cpu().numpy(), held[i][j]), (step, i, key)
                assert np.array_equal(st[key + "_scale"].cpu().numpy(), scales[i][j]), (step, i, key)


def test_held_averages_follow_the_true_ones():
    """A second moment whose gradient shrinks tenfold: its held root follows the decay (to nearest it would stand still).  The remainder
    lottery leaves an element within some 25 % of its mean; the mean of 64 K elements within 5 x 0.25 / 256."""
    count = 1 << 16
    p = torch.nn.Parameter(torch.zeros(count, device=DEV))
    opt = FusedAdamW([p], lr=0.0, weight_decay=0.0, state_bits=8)
    scale = torch.ones(count, device=DEV)
    scale[::256] = 8.0                                           # (each block's maximum: held exactly)
    r2 = 0.0
    for step in range(1500):
        size = 1.0 if step < 500 else 0.1
        p.grad = size * scale
        opt.step()
        r2 = 0.999 * r2 + 0.001 * size ** 2
    st = opt.state[p]
    root = st["exp_avg_sq_root"].float() * st["exp_avg_sq_root_scale"].repeat_interleave(256)
    inner = torch.arange(count, device=DEV) % 256 != 0
    second = float(root[inner].square().mean())
    assert abs(second / r2 - 1) < 0.1, (second, r2)              # (E r^2 = r^2 (1 + 0.2^2) with the lottery's spread)
    m = st["exp_avg"].float() * st["exp_avg_scale"].repeat_interleave(256)
    assert abs(float(m[inner].mean()) / 0.1 - 1) < 0.02


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite_stay_where_they_are(bits):
    p = torch.nn.Parameter(torch.ones(1024, device=DEV))
    opt = FusedAdamW([p], state_bits=bits, lr=1e-3)
    p.grad = torch.full((1024,), 0.01, device=DEV)
    opt.step()
    p.grad[5], p.grad[300], p.grad[700] = float("nan"), float("inf"), -float("inf")
    opt.step()
    opt.step()
    lost = torch.zeros(1024, dtype=torch.bool, device=DEV)
    lost[[5, 300, 700]] = True
    assert not torch.isfinite(p[lost]).any() and torch.isfinite(p[~lost]).all()
    q = torch.nn.Parameter(torch.ones(1024, device=DEV))
    ref = FusedAdamW([q], state_bits=bits, lr=1e-3)
    q.grad = torch.full((1024,), 0.01, device=DEV)
    for _ in range(3):
        ref.step()
    assert torch.equal(p[~lost], q[~lost])


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_tiny_ones(bits):
    """All moments 0: nothing but the decay happens.  Gradients whose squares vanish in fp32 do not divide by zero."""
    p = torch.nn.Parameter(torch.ones(600, device=DEV))
    opt = FusedAdamW([p], lr=0.5, weight_decay=0.1, state_bits=bits)
    p.grad = torch.zeros(600, device=DEV)
    opt.step()
    assert torch.equal(p.detach(), torch.full((600,), float(np.float32(0.95)), device=DEV))
    p.grad = torch.full((600,), 1e-30, device=DEV)
    opt.step()
    assert torch.isfinite(p).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_late_and_missing_gradients(bits):
    """Empty tensors, tensors without a gradient, one that joins a step later, two groups, more tensors than one launch takes."""
    gen = torch.Generator().manual_seed(5)
    params = parameters([17] * 60, torch.float32, gen) + [torch.nn.Parameter(torch.zeros(0, device=DEV))] + parameters([300, 300], torch.bfloat16, gen)
    opt = FusedAdamW([dict(params=params[:40], weight_decay=0.0), dict(params=params[40:], lr=1e-2)], lr=1e-3, state_bits=bits)
    alone = [torch.nn.Parameter(p.detach().clone()) for p in params]
    singles = [FusedAdamW([q], lr=1e-3 if i < 40 else 1e-2, weight_decay=0.0 if i < 40 else 1e-2, state_bits=bits, seed=i) for i, q in enumerate(alone)]
    for step in range(3):
        gradients(params, gen)
        params[3].grad = None
        if step == 0:
            params[50].grad = None
        for p, q, o in zip(params, alone, singles):
            q.grad = None if p.grad is None else p.grad.clone()
            o.step()
        opt.step()
    for i, (p, q) in enumerate(zip(params, alone)):
        assert torch.equal(p.detach(), q.detach()), i
    assert not opt.state[params[3]] and int(opt.state[params[50]]["step"]) == 2


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints(bits, dtype):
    """A restored optimizer goes on bit for bit; moments keep their types; other widths are refused."""
    gen = torch.Generator().manual_seed(6)
    params = parameters([1000, 77], DTYPES[dtype], gen)
    opt = FusedAdamW(params, state_bits=bits, seed=9, **HYPER)
    gradients(params, gen)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = FusedAdamW(twins, state_bits=bits, **HYPER)
    other.load_state_dict(saved)
    for p in params:
        for key, v in opt.state[p].items():
            if key != "step":
                assert v.dtype == (torch.float8_e4m3fn if bits == 8 and not key.endswith("_scale") else torch.float32)
    for _ in range(2):
        gradients(params, gen)
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        opt.step()
        other.step()
    for p, q in zip(params, twins):
        assert torch.equal(p.detach(), q.detach())
        for a, b in zip(opt.state[p].values(), other.state[q].values()):
            assert (a == b) if isinstance(a, int) else torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    with pytest.raises(ValueError):
        FusedAdamW(twins, state_bits=40 - bits).load_state_dict(saved)


def test_agrees_with_torch_over_many_steps():
    """50 steps beside torch.optim.AdamW in 64 bits: the accumulated roundings of 50 updates of at most lr, 8 x 50 u each, and of p itself."""
    gen = torch.Generator().manual_seed(8)
    params = parameters([500], torch.float32, gen)
    ref = [torch.nn.Parameter(params[0].detach().cpu().double())]
    a, b = FusedAdamW(params, **HYPER), torch.optim.AdamW(ref, **HYPER)
    for _ in range(50):
        gradients(params, gen)
        ref[0].grad = params[0].grad.cpu().double()
        a.step()
        b.step()
    off = (params[0].detach().cpu().double() - ref[0].detach()).abs()
    assert bool((off <= 50 * 2.0 ** -24 * (ref[0].detach().abs() + 0.05) + 50 * HYPER["lr"] * 400 * 2.0 ** -24).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_steps(bits):
    """factors from device memory: a step recorded once and replayed with new gradients and a moving rate, eager work between."""
    gen = torch.Generator().manual_seed(10)
    params = parameters([3000, 50], torch.float32, gen)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt, ref = (FusedAdamW(q, state_bits=bits, **HYPER) for q in (params, twins))
    import ctypes as C

    from freesound_classification_amd import _lib
    from freesound_classification_amd.ops.training import _lib as same
    assert same is _lib
    gradients(params, gen)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    opt.step()
    ref.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    factors = torch.zeros(4, device=DEV)
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        opt.factors_dev = factors
        with torch.cuda.graph(graph, stream=side):
            opt.step()
        opt.factors_dev = None
        for step, lr in ((2, 1e-3), (3, 5e-3), (4, 2e-3)):
            buf = (C.c_float * 4)()
            _lib.load().fsc_adamw_step_factors(lr, 0.9, 0.999, 0.1, step, buf)
            factors.copy_(torch.tensor(list(buf)))
            for p, q in zip(params, twins):
                g = torch.randn(p.shape, generator=gen).to(DEV)
                p.grad.copy_(g)
                q.grad.copy_(g)
            ref.param_groups[0]["lr"] = lr
            graph.replay()
            ref.step()
            torch.cuda.synchronize()
            for p, q in zip(params, twins):
                assert torch.equal(p.detach(), q.detach()), step
                for key in opt._keys():
                    assert torch.equal(opt.state[p][key].view(torch.uint8), ref.state[q][key].view(torch.uint8)), (step, key)


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(8, 8, device=DEV).t())
    p.grad = torch.zeros_like(p)
    with pytest.raises(FscError):
        FusedAdamW([p]).step()
    q = torch.nn.Parameter(torch.zeros(8, device=DEV, dtype=torch.float64))
    q.grad = torch.zeros_like(q)
    with pytest.raises(FscError):
        FusedAdamW([q]).step()
    r = torch.nn.Parameter(torch.zeros(8, 3, device=DEV))
    r.grad = torch.zeros(8, 3, device=DEV).to_sparse()
    with pytest.raises(RuntimeError):
        FusedAdamW([r]).step()


@pytest.mark.parametrize("bits", [32, 8])
def test_refusals_after_a_step(bits):
    """Moments of another size or device than the parameter's, a gradient of another type, a plain recording: refused, and nothing changes."""
    p = torch.nn.Parameter(torch.ones(600, device=DEV))
    p.grad = torch.ones_like(p)
    opt = FusedAdamW([p], state_bits=bits)
    opt.step()
    held = {key: value for key, value in opt.state[p].items()}
    before = p.detach().clone()

    def refused():
        with pytest.raises(FscError):
            opt.step()
        assert torch.equal(p.detach(), before) and opt.state[p]["step"] == 1

    opt.state[p]["exp_avg"] = held["exp_avg"].cpu()
    refused()
    opt.state[p]["exp_avg"] = held["exp_avg"][:599]
    refused()
    opt.state[p]["exp_avg"] = held["exp_avg"]
    grad = p.grad
    p.grad = None
    p.grad_dtype = torch.bfloat16
    p.grad = torch.ones(600, device=DEV, dtype=torch.bfloat16)
    refused()
    p.grad = None
    p.grad_dtype = torch.float32
    p.grad = grad
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph, other = torch.cuda.CUDAGraph(), torch.zeros(8, device=DEV)
        with torch.cuda.graph(graph, stream=stream):
            other.add_(1.0)
            refused_here = False
            try:
                opt.step()
            except FscError:
                refused_here = True
    torch.cuda.synchronize()
    assert refused_here and torch.equal(p.detach(), before) and opt.state[p]["step"] == 1
    opt.step()
    assert opt.state[p]["step"] == 2 and not torch.equal(p.detach(), before)
