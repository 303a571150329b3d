"""AdamW on the device: what a recorded training step leaves behind on the host."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

from freesound_classification_amd._lib import FscError  # noqa: E402
from freesound_classification_amd.ops.training import CapturedTrainingStep, FusedAdamW  # noqa: E402

DEV = "cuda:0"


class Tiny(torch.nn.Module):
    """What CapturedTrainingStep needs of a model: here (x shape * weight + bias - y)^2, three parameters (`spare`: the shape is not used)."""

    spare = False

    def __init__(self, bits):
        super().__init__()
        gen = torch.Generator().manual_seed(7)
        self.shape, self.weight, self.bias = (torch.nn.Parameter(torch.randn(300, generator=gen).to(DEV)) for _ in range(3))
        self.optimizer = FusedAdamW([dict(params=[self.shape, self.weight]), dict(params=[self.bias], weight_decay=0.0)], lr=1e-2, state_bits=bits)
        self._reducer = None
        self.config = types.SimpleNamespace(train=types.SimpleNamespace(accumulation_steps=1), network=types.SimpleNamespace(output_dropout=0.0))

    def training_step(self, x, y):
        off = (x if self.spare else x * self.shape) * self.weight + self.bias - y
        loss = (off * off).mean()
        loss.backward()
        self.optimizer.step()
        self.optimizer.zero_grad()
        return off.detach(), (off * off).detach(), loss.detach()


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_mark_what_they_change(bits):
    """A graph of a weight kept over a replay must notice the change, as over an eager step."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, y = (torch.randn(300, generator=gen, device=DEV) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model = Tiny(bits)
        model.training_step(x, y)
        step = CapturedTrainingStep(model, x, y)
        for _ in range(2):
            tensors = list(model.parameters()) + [v for p in model.parameters() for k, v in model.optimizer.state[p].items() if k != "step"]
            seen = [t._version for t in tensors]
            late = model.weight.square().sum()
            step(x, y)
            assert all(t._version > v for t, v in zip(tensors, seen))
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                late.backward()
    torch.cuda.synchronize()


@pytest.mark.parametrize("spare", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_at_rest_keeps_its_step_count(bits, spare):
    """A parameter, first in the optimizer, that was trained for two steps and then frozen, or that the recorded step (the sixth) does not use: a
    recording of the others goes on from their step count, not from its, and leaves it alone.  The same updates as eager ones, bit for bit."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    x, y = (torch.randn(300, generator=gen, device=DEV) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        models = [Tiny(bits), Tiny(bits)]
        for model in models:
            for i in range(5):
                model.shape.requires_grad_(spare or i < 2)
                model.training_step(x, y)
            model.spare = spare
        step = CapturedTrainingStep(models[0], x, y)
        for count in (6, 7, 8):
            step(x, y)
            models[1].training_step(x, y)
            for a, b in zip(models[0].parameters(), models[1].parameters()):
                assert torch.equal(a.detach(), b.detach())
            for model in models:
                assert [int(model.optimizer.state[p]["step"]) for p in model.parameters()] == [5 if spare else 2, count, count]
    torch.cuda.synchronize()


@pytest.mark.parametrize("change", ["checkpoint", "moment", "weight"])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_recording_of_other_tensors_is_refused(bits, change):
    """The recorded step writes where parameters and moments were: once they have been replaced (and the old ones may be somebody else's memory), it is
    not replayed.  A checkpoint of the model, which is copied into place, is fine."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    x, y = (torch.randn(300, generator=gen, device=DEV) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model = Tiny(bits)
        model.training_step(x, y)
        step = CapturedTrainingStep(model, x, y)
        step(x, y)
        model.load_state_dict({k: v.clone() for k, v in model.state_dict().items()})
        step(x, y)
        step.sync_state()
        kept = model.weight.data, model.optimizer.state[model.weight]["exp_avg"]          # (so that the recording's memory stays what it was)
        if change == "checkpoint":
            old = [dict(st) for st in model.optimizer.state.values()]
            model.optimizer.load_state_dict(model.optimizer.state_dict())
            assert len(old) == 3
        elif change == "moment":
            model.optimizer.state[model.weight]["exp_avg"] = kept[1].clone()
        else:
            model.weight.data = kept[0].clone()
        before = model.weight.detach().clone()
        with pytest.raises(FscError, match="record the step again"):
            step(x, y)
        assert torch.equal(model.weight.detach(), before) and int(model.optimizer.state[model.weight]["step"]) == 3
        again = CapturedTrainingStep(model, x, y)
        again(x, y)
        assert not torch.equal(model.weight.detach(), before) and int(model.optimizer.state[model.weight]["step"]) == 4
    torch.cuda.synchronize()


def test_held_moments_are_right_in_the_mean():
    """64 K elements beside one that is 9.3 times theirs in each block of 256 (the block's maximum: held exactly, as its scale), whose gradients then
    fall tenfold.

    The first moment is linear in what is held and rounding is right in the mean, so its mean is the true one within 5 deviations of a mean over the
    elements.  The root: a step takes r to sqrt(beta2 r^2 + ...), which is convex, so a spread of s (relative to the mean) lifts the mean by s^2 / 2 at
    most.  The spread: a code that falls by d is rounded to one of its neighbours, D apart, with a variance of d D; over a fall from code c0 to c1 that
    is s^2 = the integral of (D / c) dlog(c), with 1/16 <= D / c <= 1/8 where codes are normal (above 2^-6), on top of what was there.  The second moment
    that a step starts from is the root's square, so in the mean it is above the true one by that s^2: it is not right in the mean, the root is."""
    count, steps = 1 << 16, (1000, 1500, 2500)
    p = torch.nn.Parameter(torch.zeros(count, device=DEV))
    opt = FusedAdamW([p], lr=0.0, weight_decay=0.0, state_bits=8, seed=5)
    inner = torch.arange(count, device=DEV) % 256 != 0
    many = int(inner.sum())
    m = v = top = 0.0
    was = None
    for step in range(1, steps[-1] + 1):
        g = 1.0 if step <= steps[0] else 0.1
        p.grad = torch.where(inner, g, 9.3)
        opt.step()
        m, v, top = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g, 0.999 * top + 0.001 * 9.3 ** 2
        if step not in steps:
            continue
        st = opt.state[p]
        held = (st["exp_avg"].float() * st["exp_avg_scale"].repeat_interleave(256))[inner].double()
        assert abs(float(held.mean()) - m) <= 5 * float(held.std()) / many ** 0.5
        root = (st["exp_avg_sq_root"].float() * st["exp_avg_sq_root_scale"].repeat_interleave(256))[inner].double()
        mean, code = float(root.mean()), 448 * (v / top) ** 0.5
        spread2 = float(root.var()) / mean ** 2
        luck = 5 * (spread2 / many) ** 0.5
        assert abs(mean / v ** 0.5 - 1) <= spread2 / 2 + luck, (step, mean / v ** 0.5)
        if was is None:
            was = spread2, code
            assert spread2 < 1 / 8 ** 2 and code > 32                # (at rest between two neighbours at most 1 / 8 apart)
        else:
            fall = torch.log(torch.tensor(was[1] / code)).item()
            few = 5 * (2 / many) ** 0.5 * spread2                   # (of an estimated variance)
            assert fall / 16 - few <= spread2 <= was[0] + fall / 8 + few, (step, spread2, fall)
        excess = float(root.square().mean()) / v - 1
        assert abs(excess - spread2) <= (spread2 + 2 * luck) * (1 + spread2), (step, excess)
