"""AdamW's host side without a device: what a step looks at before it launches.  The launch itself is replaced by one that notes its table;
tensors in host memory stand for those of device 0."""
import copy
import ctypes as C
import io

import numpy as np
import pytest
import torch

from freesound_classification_amd import _lib
from freesound_classification_amd.networks.classifiers import SsmHead
from freesound_classification_amd.ops import training
from freesound_classification_amd.ops.training import FusedAdamW


@pytest.fixture
def launches(monkeypatch):
    """Every launch: (rows of the tensor table, arguments)."""
    made = []

    def note(name, table, n, *args):
        made.append((np.ctypeslib.as_array(C.cast(table, C.POINTER(C.c_int64)), (n, 8)).copy(), args))

    elsewhere = set()
    monkeypatch.setattr(training, "call", note)
    monkeypatch.setattr(training, "stream_ptr", lambda: 0)
    monkeypatch.setattr(training, "_device_number", lambda t: 1 if id(t) in elsewhere else 0)
    monkeypatch.setattr(_lib, "_get_device", lambda: 0)
    made_on = made, elsewhere
    return made_on


def _parameters(*sizes, dtype=torch.float32):
    params = [torch.nn.Parameter(torch.ones(size, dtype=dtype)) for size in sizes]
    for p in params:
        p.grad = torch.ones_like(p)
    return params


KEYS = {32: ["exp_avg", "exp_avg_sq"], 8: ["exp_avg", "exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale"]}


def _wrong(good):
    """What must not be launched in the place of a good moment: another size, another type, strides, not a tensor, nothing."""
    n = good.numel()
    other = torch.bfloat16 if good.dtype == torch.float32 else torch.uint8
    wide = torch.zeros(2 * n, dtype=good.dtype)
    return [good[:n - 1], torch.zeros(n + 1, dtype=good.dtype), torch.zeros(n, dtype=other), torch.zeros(n, dtype=torch.float64), wide[::2],
            torch.zeros(1, dtype=good.dtype).expand(n), good.numpy(force=True) if good.dtype == torch.float32 else None, None]


@pytest.mark.parametrize("bits, key", [(bits, key) for bits in (32, 8) for key in KEYS[bits]])
def test_every_moment_is_looked_at(launches, bits, key):
    made, elsewhere = launches
    params = _parameters(600, 300)
    opt = FusedAdamW(params, state_bits=bits)
    opt.step()
    assert len(made) == 1 and made[0][0][:, 6].tolist() == [600, 300]
    st = opt.state[params[0]]
    held = [opt.state[p][k].data_ptr() for p in params for k in KEYS[bits]]
    assert made[0][0][:, 2:2 + len(KEYS[bits])].reshape(-1).tolist() == held
    good = st[key]
    for bad in _wrong(good):
        st[key] = bad
        with pytest.raises(_lib.FscError, match="moments"):
            opt.step()
    del st[key]
    with pytest.raises(_lib.FscError, match="moments"):
        opt.step()
    st[key] = good
    elsewhere.add(id(good))
    with pytest.raises(_lib.FscError, match="device"):
        opt.step()
    elsewhere.clear()
    assert len(made) == 1 and all(opt.state[p]["step"] == 1 for p in params)
    opt.step()
    assert len(made) == 2 and all(opt.state[p]["step"] == 2 for p in params)


@pytest.mark.parametrize("bits", [32, 8])
def test_no_moments_are_made_where_others_are_refused(launches, bits):
    made, _ = launches
    params = _parameters(600, 300)
    params[1].grad = None
    opt = FusedAdamW(params, state_bits=bits)
    opt.step()
    params[1].grad = torch.ones(300)
    opt.state[params[0]]["exp_avg"] = torch.zeros(599)
    with pytest.raises(_lib.FscError, match="moments"):
        opt.step()
    assert not opt.state[params[1]] and len(made) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_late_parameters_and_types_get_their_own_launches(launches, bits):
    """What the table of a launch holds: tensors of one type and step count each, with their own moments and salts."""
    made, _ = launches
    params = _parameters(10, 20) + _parameters(30, dtype=torch.bfloat16) + _parameters(0, 513)
    params[1].grad = None
    opt = FusedAdamW(params, state_bits=bits, seed=5)
    opt.step()
    params[1].grad = torch.ones(20)
    opt.step()
    tables = [sorted(zip(t[:, 6].tolist(), t[:, 7].tolist())) for t, _ in made]
    assert tables == [[(0, 8), (10, 5), (513, 9)], [(30, 7)], [(0, 8), (10, 5), (513, 9)], [(20, 6)], [(30, 7)]]
    for table, _ in made[2:]:
        for row in table:
            p = next(p for p in params if p.numel() == row[6])
            assert row[:2 + len(KEYS[bits])].tolist() == [p.data_ptr(), p.grad.data_ptr()] + [opt.state[p][k].data_ptr() for k in KEYS[bits]]
    assert [opt.state[p]["step"] for p in params] == [2, 1, 2, 2, 2]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_checkpoint_changes_nothing(launches, bits, dtype):
    """One moment of another shape or missing, an 8-bit one in another type, no step count, other groups: the optimizer stays as it was."""
    params = _parameters(8, 300, dtype=dtype)
    opt = FusedAdamW(params, state_bits=bits, seed=3)
    opt.step()
    before = [dict(opt.state[p]) for p in params]
    good = {"state": {i: dict(opt.state[p]) for i, p in enumerate(params)}, "param_groups": [dict(opt.param_groups[0], params=[0, 1], lr=0.5)],
            "state_bits": bits, "seed": 4}

    def damaged(change):
        out = dict(good, state={i: dict(st) for i, st in good["state"].items()}, param_groups=[dict(good["param_groups"][0])])
        change(out)
        return out

    bad = [damaged(lambda c, key=key: c["state"][1].update({key: c["state"][1][key][:-1]})) for key in KEYS[bits]]
    bad += [damaged(lambda c, key=key: c["state"][1].pop(key)) for key in KEYS[bits] + ["step"]]
    bad += [damaged(lambda c: c["param_groups"][0].update(params=[0])), damaged(lambda c: c.update(state_bits=40 - bits)),
            damaged(lambda c: c["param_groups"].append(dict(c["param_groups"][0])))]
    if bits == 8:
        bad.append(damaged(lambda c: c["state"][1].update(exp_avg=c["state"][1]["exp_avg"].float())))
    for checkpoint in bad:
        with pytest.raises(ValueError):
            opt.load_state_dict(checkpoint)
        assert opt.seed == 3 and opt.param_groups[0]["lr"] == 1e-3
        for p, held in zip(params, before):
            assert opt.state[p].keys() == held.keys() and all(opt.state[p][key] is held[key] for key in held)
    opt.load_state_dict(good)
    assert opt.seed == 4 and opt.param_groups[0]["lr"] == 0.5
    for p, held in zip(params, before):
        for key in KEYS[bits]:
            assert opt.state[p][key] is not held[key] and opt.state[p][key].dtype == held[key].dtype
            assert torch.equal(opt.state[p][key].view(torch.uint8), held[key].view(torch.uint8))
        assert opt.state[p]["step"] == 1
    opt.step()
    assert opt.state[params[0]]["step"] == 2


@pytest.mark.parametrize("option", ["amsgrad", "maximize"])
def test_options_that_change_the_rule_are_refused(option):
    """torch.optim.AdamW's checkpoints carry them, and a group may: neither is dropped in silence.  Options that are off pass."""
    p, q = _parameters(4, 4)
    ref = torch.optim.AdamW([torch.nn.Parameter(torch.ones(4))], **{option: True})
    opt = FusedAdamW([p], lr=0.25)
    with pytest.raises(ValueError, match=option):
        opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 0.25
    with pytest.raises(ValueError, match=option):
        opt.add_param_group({"params": [q], option: True})
    with pytest.raises(ValueError, match=option):
        FusedAdamW([{"params": [p], option: True}])
    assert len(opt.param_groups) == 1
    opt.load_state_dict(torch.optim.AdamW([torch.nn.Parameter(torch.ones(4))], lr=0.125).state_dict())
    opt.add_param_group({"params": [q], option: False})
    assert opt.param_groups[0]["lr"] == 0.125 and len(opt.param_groups) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_marks_what_it_changes(launches, bits):
    """A graph that saved a weight (or a moment) must notice that a step has changed it; a parameter without a gradient is not touched."""
    p, q = _parameters(5, 5)
    q.grad = None
    opt = FusedAdamW([p, q], state_bits=bits)
    opt.step()
    seen = [p._version, q._version] + [opt.state[p][key]._version for key in KEYS[bits]]
    squares, others = p.square().sum(), q.square().sum()
    scaled = None
    if bits == 32:
        scaled = (torch.ones(5, requires_grad=True) * opt.state[p]["exp_avg_sq"]).sum()
    opt.step()
    assert [p._version, q._version] + [opt.state[p][key]._version for key in KEYS[bits]] == [seen[0] + 1, seen[1]] + [v + 1 for v in seen[2:]]
    for late in [squares] + ([scaled] if bits == 32 else []):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            late.backward()
    others.backward()


def _saved(opt):
    """Through torch's pickle (the bare one cannot read e4m3 tensors back)."""
    file = io.BytesIO()
    torch.save(opt, file)
    file.seek(0)
    return torch.load(file, weights_only=False)


@pytest.mark.parametrize("copied", [copy.deepcopy, _saved])
@pytest.mark.parametrize("bits", [32, 8])
def test_copies_of_the_optimizer(launches, bits, copied):
    """A copy holds its moments in the same width, goes on with the same random numbers and the same scale, and has a step of its own."""
    made, _ = launches
    (p,) = _parameters(300)
    opt = FusedAdamW([p], lr=0.5, state_bits=bits, seed=11)
    opt.grad_scale = 0.25
    opt.step()
    opt.factors_dev = torch.zeros(4)                         # (of a recording that is being made: not the copy's)
    twin = copied(opt)
    assert (twin.state_bits, twin.seed, twin.grad_scale, twin.factors_dev) == (bits, 11, 0.25, None)
    (q,) = twin.param_groups[0]["params"]
    assert q is not p and twin.state[q]["step"] == 1 and twin.param_groups[0]["lr"] == 0.5
    opt.factors_dev = None
    for o, leaf in ((opt, p), (twin, q)):
        leaf.grad = torch.ones_like(leaf)
        o.step()
    assert made[1][0][0, 7] == made[2][0][0, 7] == 11 and made[2][0][0, 0] == q.data_ptr() and made[1][1][-2] == made[2][1][-2] == 0.25
    assert twin.state_dict()["state_bits"] == bits and twin.state_dict()["seed"] == 11


@pytest.mark.parametrize("copied", [copy.deepcopy, _saved])
def test_a_copied_head_keeps_its_time_constants_out_of_the_decay(copied):
    model = torch.nn.Sequential(torch.nn.Linear(3, 4), SsmHead(6))
    for module in (model, copied(model)):
        opt = training.make_optimizer("adamw", module, 1e-3, 0.1)
        rates = {id(p): group["weight_decay"] for group in opt.param_groups for p in group["params"]}
        held = {name for name, p in module.named_parameters() if rates[id(p)] == 0.0}
        assert held == {"0.bias", "1.norm.weight", "1.norm.bias", "1.in_proj.bias", "1.conv_bias", "1.dt_proj.bias", "1.a_log", "1.d"}
