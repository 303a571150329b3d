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
