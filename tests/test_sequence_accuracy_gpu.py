"""How near the sequence kernels come to the 64-bit recurrences, measured against what plain fp32 loses on the same inputs.

Tolerances.  The plain recurrence in fp32 (oracle/sequence.py on fp32 tensors) and the kernels round the same terms as often; the kernels' exponentials,
logarithms and reciprocals are good to a unit in the last place where the plain ones are to half a unit or little more, a factor of 2, and their sums run
in another order, another 2 for luck: the 2-norm of a kernel's error is at most 4 times the plain fp32 error's, and 8 roundings (u = 2^-24) of the
result's own 2-norm, for results that the plain form happens to hit.  A 16-bit output adds its one rounding, at most eps / 2 of the result.
(Every tensor compared has 64 values at least, so that the norms are not a matter of luck.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

from freesound_classification_amd import functional as F  # noqa: E402
from oracle import sequence as oseq  # noqa: E402

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def near(got, want, plain, what):
    got, want, plain = got.detach().cpu(), want.detach(), plain.detach().double()
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    off, size, loss = float((got.double() - want).norm()), float(want.norm()), float((plain - want).norm())
    assert off <= 4 * loss + (8 * U + half) * size, "%s: %.3g of the norm, plain fp32 %.3g" % (what, off / size, loss / size)


def both(ofn, p, cot):
    """Outputs and gradients of the recurrence in 64 and in 32 bits."""
    sides = []
    for dtype in (torch.float64, torch.float32):
        leaves = {k: v.to(dtype).requires_grad_() for k, v in p.items()}
        out = ofn(leaves)
        sides.append(list(out) + list(torch.autograd.grad(out, list(leaves.values()), [c.to(dtype) for c in cot])))
    return sides


def kernels(fn, p, cot):
    leaves = {k: v.to(DEV).requires_grad_() for k, v in p.items()}
    out = fn(leaves)
    return list(out) + list(torch.autograd.grad(out, list(leaves.values()), [c.to(DEV) for c in cot]))


def scan_case(n, t, d, s, g, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    rate = torch.exp(torch.rand(d, generator=gen) * 4.6 - 6.9)
    p = dict(u=randn(n, t, d).to(dtype), dt=(0.5 * randn(n, t, d)).to(dtype), a_log=torch.log(torch.arange(1, s + 1).float()).repeat(d, 1) + 0.2 * randn(d, s),
             b=randn(n, t, g, s).to(dtype), c=randn(n, t, g, s).to(dtype), d=randn(d), z=randn(n, t, d).to(dtype),
             dt_bias=rate + torch.log(-torch.expm1(-rate)), initial=randn(n, d, s))
    lengths = [t] + [max(1, t * (i + 1) // (n + 1)) for i in range(n - 1)]
    return p, lengths, (randn(n, t, d).to(dtype), randn(n, d, s))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n, t, d, s, g", [
    (2, 53, 96, 16, 1), (3, 40, 70, 5, 2), (1, 431, 128, 16, 1), (2, 333, 72, 20, 2), (1, 260, 64, 64, 1), (2, 700, 64, 3, 1), (1, 900, 66, 8, 3)])
def test_selective_scan(n, t, d, s, g, dtype):
    """Whole sequences and, from 260 frames on, time cut into segments; ragged, continued, every gradient."""
    p, lengths, cot = scan_case(n, t, d, s, g, DTYPES[dtype], t + s)
    dl = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = kernels(lambda q: F.selective_scan(q["u"], q["dt"], q["a_log"], q["b"], q["c"], d=q["d"], z=q["z"], dt_bias=q["dt_bias"], lengths=dl,
                                             initial=q["initial"], return_final=True), p, cot)
    want, plain = both(lambda q: oseq.selective_scan(q["u"], q["dt"], q["a_log"], q["b"], q["c"], q["d"], q["z"], q["dt_bias"], True, lengths,
                                                     q["initial"]), p, cot)
    for name, a, b, c in zip(["y", "final"] + ["d" + k for k in p], got, want, plain):
        near(a, b, c, name)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n, t, d, k", [(3, 53, 96, 4), (2, 700, 70, 3), (1, 130, 64, 8), (4, 20, 129, 2)])
def test_causal_conv(n, t, d, k, dtype):
    gen = torch.Generator().manual_seed(t)
    randn = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    dt = DTYPES[dtype]
    p = dict(x=randn(n, t, d).to(dt), weight=randn(d, k), bias=randn(d), initial=randn(n, k - 1, d).to(dt))
    cot = randn(n, t, d).to(dt), randn(n, k - 1, d).to(dt)
    lengths = [t] + [max(1, t * (i + 1) // (n + 1)) for i in range(n - 1)]
    dl = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = kernels(lambda q: F.causal_conv(q["x"], q["weight"], q["bias"], lengths=dl, initial=q["initial"], return_final=True), p, cot)
    want, plain = both(lambda q: oseq.causal_conv(q["x"], q["weight"], q["bias"], True, lengths, q["initial"]), p, cot)
    for name, a, b, c in zip(["y", "final"] + ["d" + key for key in p], got, want, plain):
        near(a, b, c, name)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n, d, s, g", [(3, 70, 16, 2), (2, 66, 5, 1), (4, 64, 64, 1), (2, 80, 30, 4), (300, 130, 16, 1)])
def test_scan_frames_one_by_one(n, d, s, g, dtype):
    p, _, _ = scan_case(n, 9, d, s, g, DTYPES[dtype], d)
    q = {k: v.to(DEV) for k, v in p.items()}
    state = q["initial"].clone()
    got = torch.stack([F.selective_scan_step(q["u"][:, i], q["dt"][:, i], q["a_log"], q["b"][:, i], q["c"][:, i], state, d=q["d"], z=q["z"][:, i],
                                             dt_bias=q["dt_bias"]) for i in range(9)], 1)
    sides = []
    for kind in (torch.float64, torch.float32):
        r = {k: v.to(kind) for k, v in p.items()}
        sides.append(oseq.selective_scan(r["u"], r["dt"], r["a_log"], r["b"], r["c"], r["d"], r["z"], r["dt_bias"], True, None, r["initial"]))
    for name, a, b, c in zip(("y", "state"), (got, state), *sides):
        near(a, b, c, name)


@pytest.mark.parametrize("activation", ["silu", None])
@pytest.mark.parametrize("n, d, k", [(1, 1, 1), (3, 7, 4), (48, 1536, 4), (2, 24, 8)])
def test_conv_frames_one_by_one_in_fp16(n, d, k, activation):
    """Single frames give the sequence's values bit for bit (the same products in the same order), in fp16 as in the other types."""
    gen = torch.Generator(device=DEV).manual_seed(d)
    x, w, b = (torch.randn(*shape, generator=gen, device=DEV) for shape in ((n, 11, d), (d, k), (d,)))
    x = x.half()
    whole, last = F.causal_conv(x, w, b, activation=activation, return_final=True)
    y, window = F.causal_conv(x[:, :6], w, b, activation=activation, return_final=True)
    parts = [y] + [F.causal_conv_step(x[:, i], window, w, b, activation=activation)[:, None] for i in range(6, 11)]
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(window, last)
