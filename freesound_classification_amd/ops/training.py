"""Counterpart of the reference's ops/training.py: `OPTIMIZERS`, `make_scheduler`, `make_step`,
`OneCycleScheduler` with the same descriptors ("steplr_{step}_{gamma}", "1cycle_{min}_{max}").
The optimizers are fused multi-tensor HIP kernels with torch-compatible state dicts.
"""
import ctypes as C
import gc
import itertools
import operator
import os
import warnings
from functools import partial

import numpy as np
import torch
from torch.optim import Optimizer
from torch.optim.lr_scheduler import StepLR

from .. import _lib
from .._lib import OptTensor, call, stream_ptr


def _forget_packed_weights():
    # the kernels below update the weights through raw pointers (no tensor version bump): packed copies kept for inference go
    from .. import functional
    functional.forget_packed_weights()


def _table(entries):
    arr = (OptTensor * len(entries))()
    for i, (p, g, s0, s1, s2) in enumerate(entries):
        arr[i] = OptTensor(p.data_ptr(), g.data_ptr(), s0.data_ptr(),
                           s1.data_ptr() if s1 is not None else None,
                           s2.data_ptr() if s2 is not None else None, p.numel())
    return arr


def _checked_grad(p):
    g = p.grad
    if g.is_sparse:
        raise RuntimeError("sparse gradients are not supported")
    if not p.is_cuda:
        raise _lib.FscError("fused optimizers need device parameters (no CPU fallback)")
    if not g.is_contiguous():
        g = g.contiguous()
        p.grad = g
    return g


class FusedAdam(Optimizer):
    """torch.optim.Adam semantics (L2 weight decay, optional amsgrad) in one kernel per 64
    tensors.  State keys match torch (step, exp_avg, exp_avg_sq, max_exp_avg_sq).
    `grad_scale` multiplies gradients first (1/world_size after a summing all-reduce)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, amsgrad=False):
        if not amsgrad:
            raise NotImplementedError("the accelerated path ships Adam with amsgrad=True only "
                                      "(reference ops/training.py:10)")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad))
        self.grad_scale = 1.0
        self.factors_dev = None      # set while a step is recorded into a HIP graph (CapturedTrainingStep): lr / step from device memory

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        _forget_packed_weights()
        for group in self.param_groups:
            entries = []
            step = None
            for p in group["params"]:
                if p.grad is None:
                    continue
                g = _checked_grad(p)
                st = self.state[p]
                if not st:
                    st["step"] = 0
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                    st["max_exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                st["step"] = int(st["step"]) + 1
                if step is None:
                    step = st["step"]
                if st["step"] != step:       # tensors that joined late get their own launch
                    self._launch(group, [(p, g, st["exp_avg"], st["exp_avg_sq"], st["max_exp_avg_sq"])], st["step"])
                    continue
                entries.append((p, g, st["exp_avg"], st["exp_avg_sq"], st["max_exp_avg_sq"]))
            if entries:
                self._launch(group, entries, step)
        return loss

    def _launch(self, group, entries, step):
        b1, b2 = group["betas"]
        tbl = _table(entries)
        from .. import functional as F
        # reads p, g, m, v, vmax and writes p, m, v, vmax: nine fp32 streams (776 MB per step at cfg 2)
        with F._stage("optimizer", 9 * 4 * sum(e[0].numel() for e in entries)):
            if self.factors_dev is not None:
                call("fsc_adam_amsgrad_step_dev", tbl, len(entries), self.factors_dev.data_ptr(), b1, b2, group["eps"],
                     group["weight_decay"], float(self.grad_scale), stream_ptr())
            else:
                call("fsc_adam_amsgrad_step", tbl, len(entries), float(group["lr"]), b1, b2, group["eps"],
                     group["weight_decay"], int(step), float(self.grad_scale), stream_ptr())


class FusedSGD(Optimizer):
    """torch.optim.SGD(momentum, nesterov=True, dampening=0) semantics with L2 weight decay."""

    def __init__(self, params, lr, momentum=0.9, weight_decay=0.0, nesterov=True):
        if not nesterov or momentum <= 0:
            raise NotImplementedError("the accelerated path ships SGD with Nesterov momentum only "
                                      "(reference ops/training.py:11)")
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov,
                                      dampening=0))
        self.grad_scale = 1.0

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        _forget_packed_weights()
        for group in self.param_groups:
            fresh, warm = [], []
            for p in group["params"]:
                if p.grad is None:
                    continue
                g = _checked_grad(p)
                st = self.state[p]
                if "momentum_buffer" not in st or st["momentum_buffer"] is None:
                    st["momentum_buffer"] = torch.empty_like(p, memory_format=torch.contiguous_format)
                    fresh.append((p, g, st["momentum_buffer"], None, None))
                else:
                    warm.append((p, g, st["momentum_buffer"], None, None))
            for entries, first in ((fresh, 1), (warm, 0)):
                if entries:
                    call("fsc_sgd_nesterov_step", _table(entries), len(entries), float(group["lr"]),
                         group["momentum"], group["weight_decay"], first, float(self.grad_scale), stream_ptr())
        return loss


_PARAM_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# (applied with map: a step looks at every tensor of the model, and the loop in C costs half of one in Python)
_dtype_of, _grad_of = operator.attrgetter("dtype"), operator.attrgetter("grad")
_step_of = operator.itemgetter("step")
_is_none = partial(operator.is_, None)
_is_contiguous, _address, _numel, _device_number = torch.Tensor.is_contiguous, torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device
# (the kernels write through raw addresses; a graph that saved a weight in front of a step must not go on with the new one)
_mark_changed = torch.autograd.graph.increment_version
STATE_BLOCK = 256        # elements that share one scale of an 8-bit moment


class FusedAdamW(Optimizer):
    """AdamW (torch.optim.AdamW's rule: weight decay apart from the moments) over all tensors of a group in one launch per 52 tensors.

    `state_bits=32`: state keys match torch (step, exp_avg, exp_avg_sq), moments in fp32.  `state_bits=8`: the moments are held as e4m3 values
    with one fp32 scale per 256 elements -- exp_avg / exp_avg_scale, and the square root of the second moment, exp_avg_sq_root /
    exp_avg_sq_root_scale --, 2.03 bytes a parameter instead of 8, rounded stochastically: the random bits are a function of (`seed`, the
    tensor's place in the optimizer, the step, the element), so a run is reproducible.  The means of the first moment and of the root are the
    true ones; the second moment, the root's square, is above its own by the variance of the rounding (under 0.5 %, more where an element's
    gradients shrink against its neighbours').  Parameters and gradients are fp32, bf16 or fp16.
    `grad_scale` multiplies gradients first (1 / world_size after a summing all-reduce).  A refused step changes nothing in its group, a
    refused checkpoint nothing at all; a step is recorded into a HIP graph by CapturedTrainingStep alone (elsewhere the step count would be frozen into it)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8, got %r" % (state_bits,))
        if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0 and all(0.0 <= b < 1.0 for b in betas)):
            raise ValueError("FusedAdamW: lr, eps and weight_decay must be >= 0 and the betas in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits = state_bits
        self.seed = int(seed)
        self.grad_scale = 1.0
        self.factors_dev = None      # set while a step is recorded into a HIP graph: four floats a group in device memory

    def _keys(self):
        return ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("exp_avg", "exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale")

    def _new_state(self, p):
        st = {"step": 0}
        blocks = -(-p.numel() // STATE_BLOCK)
        for key in self._keys():
            st[key] = torch.zeros(blocks if key.endswith("_scale") else p.shape, device=p.device, dtype=self._held_dtype(key))
        return st

    def _held_dtype(self, key):
        return torch.float32 if self.state_bits == 32 or key.endswith("_scale") else torch.float8_e4m3fn

    @staticmethod
    def _known_options(group):
        """A group's (or a checkpoint's) options that change torch's rule into one that this optimizer does not have."""
        for option in ("amsgrad", "maximize"):
            if group.get(option):
                raise ValueError("FusedAdamW: %s is not supported" % option)

    def __getstate__(self):
        """(torch keeps defaults, state and groups alone; the width and the seed are part of what the state means)"""
        return dict(super().__getstate__(), state_bits=self.state_bits, seed=self.seed, grad_scale=self.grad_scale, factors_dev=None)

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            self._known_options(param_group)
        super().add_param_group(param_group)
        params = self.param_groups[-1]["params"]
        if len(set(map(id, params))) != len(params):         # (one launch updates them side by side: twice would be a race)
            self.param_groups.pop()
            raise ValueError("FusedAdamW: a parameter appears more than once in a group")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self.factors_dev is None and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise _lib.FscError("FusedAdamW: a recorded step would repeat this step's bias corrections; record it with CapturedTrainingStep")
        _forget_packed_weights()
        place = 0
        for gi, group in enumerate(self.param_groups):
            params, salts = group["params"], np.arange(place, place + len(group["params"]))
            place += len(params)
            grads = list(map(_grad_of, params))
            missing = list(map(_is_none, grads))
            if any(missing):
                params, salts = [p for p, none in zip(params, missing) if not none], salts[np.logical_not(missing)]
                grads = list(map(_grad_of, params))
            if not params:
                continue
            types, counts = list(map(_dtype_of, params)), list(map(_numel, params))
            grads = self._checked(params, grads, types, counts)
            states = list(map(self.state.__getitem__, params))
            if not all(states):                              # (the moments that are there are looked at before any are made)
                there = [(st, count) for st, count in zip(states, counts) if st]
                self._moments([st for st, _ in there], [count for _, count in there])
                for p, st in zip(params, states):
                    if not st:
                        st.update(self._new_state(p))
            moments = self._moments(states, counts)
            steps = list(map(_step_of, states))
            kind, *others = dict.fromkeys(zip(types, steps)) if len(set(types)) > 1 or len(set(steps)) > 1 else [(types[0], steps[0])]
            if not others:
                self._launch(gi, group, *kind, params, grads, moments, states, salts, counts)
                continue
            # one launch sequence for what shares its type and step count: all of them but for parameters that joined late
            for kind in (kind, *others):
                at = [i for i, k in enumerate(zip(types, steps)) if k == kind]
                pick = lambda values: [values[i] for i in at]  # noqa: E731
                self._launch(gi, group, *kind, pick(params), pick(grads), list(map(pick, moments)), pick(states), pick(salts), pick(counts))
        return loss

    @staticmethod
    def _checked(params, grads, types, counts):
        """The gradients, contiguous; nothing has changed yet when this refuses."""
        devices = set(map(_device_number, params + grads))
        if -1 in devices:
            raise _lib.FscError("FusedAdamW needs device parameters (no CPU fallback)")
        if devices != {_lib._get_device()}:
            raise _lib.FscError("FusedAdamW: the parameters of a group must be on the current device")
        if not _PARAM_DTYPES.keys() >= set(types):
            raise _lib.FscError("FusedAdamW: parameters are fp32, bf16 or fp16, got %s" % sorted(map(str, set(types) - _PARAM_DTYPES.keys())))
        if not all(map(_is_contiguous, params)):
            raise _lib.FscError("FusedAdamW: parameters must be contiguous")
        if not all(map(_is_contiguous, grads)):
            grads = [_checked_grad(p) for p in params]
        if list(map(_dtype_of, grads)) != types or list(map(_numel, grads)) != counts:
            raise _lib.FscError("FusedAdamW: a gradient's type or size is not its parameter's")
        return grads

    def _moments(self, states, counts):
        """The states' tensors, a list for each key.  The kernel is given their addresses alone, so every one is looked at: what a loader, a
        cast or a move has left there must be of the type, size and device that it is read and written as.  (Some 5 us for each look at 141
        tensors: 27 us of a step with 32 bits, 62 with 8.)"""
        keys = self._keys()
        try:
            held = [list(map(operator.itemgetter(key), states)) for key in keys]
            sizes = {False: list(counts), True: [-(-count // STATE_BLOCK) for count in counts]}
            sound = not states or set(map(_device_number, itertools.chain(*held))) == {_lib._get_device()}
            for key, tensors in zip(keys, held):
                sound = (sound and set(map(_dtype_of, tensors)) <= {self._held_dtype(key)} and all(map(_is_contiguous, tensors))
                         and list(map(_numel, tensors)) == sizes[key.endswith("_scale")])
        except (KeyError, TypeError, AttributeError) as e:
            raise _lib.FscError("FusedAdamW: a parameter's moments are not those of %d bits (%r)" % (self.state_bits, e)) from e
        if not sound:
            raise _lib.FscError("FusedAdamW: the moments are not on the parameters' device, or not of their size, contiguous and of the type "
                                "that %d bits are held in" % self.state_bits)
        return held

    def _launch(self, gi, group, dtype, step, tensors, grads, moments, states, salts, counts):
        step = int(step) + 1
        n = len(tensors)
        table = np.zeros((8, n), dtype=np.int64)
        for row, values in enumerate([tensors, grads, *moments]):
            table[row] = np.fromiter(map(_address, values), np.int64, n)
        table[6] = counts
        table[7] = (np.asarray(salts) + (self.seed & 0xFFFFFFFF)) & 0xFFFFFFFF
        table = np.ascontiguousarray(table.T)
        b1, b2 = group["betas"]
        factors, dev = None, None
        if self.factors_dev is not None:
            dev = self.factors_dev.data_ptr() + 16 * gi
        else:
            factors = (C.c_float * 4)()
            _lib.load().fsc_adamw_step_factors(float(group["lr"]), b1, b2, float(group["weight_decay"]), step, factors)
        from .. import functional as F
        held = 8 if self.state_bits == 32 else 2
        with F._stage("optimizer", sum(counts) * (3 * tensors[0].element_size() + 2 * held)):
            call("fsc_adamw_step", table.ctypes.data, n, _PARAM_DTYPES[dtype], self.state_bits, factors, dev, b1, b2,
                 float(group["eps"]), float(self.grad_scale), stream_ptr())
        _mark_changed(itertools.chain(tensors, *moments))
        for st in states:
            st["step"] = step

    def state_dict(self):
        out = super().state_dict()
        out["state_bits"], out["seed"] = self.state_bits, self.seed
        return out

    def load_state_dict(self, state_dict):
        """Like torch's, but the moments keep the types they are held in (torch casts floating state to the parameter's type), and a checkpoint
        that is refused leaves the optimizer as it was."""
        if state_dict.get("state_bits", 32) != self.state_bits:
            raise ValueError("FusedAdamW: the checkpoint holds its moments in %d bits, the optimizer in %d"
                             % (state_dict.get("state_bits", 32), self.state_bits))
        for group in state_dict["param_groups"]:
            self._known_options(group)
        params = [p for group in self.param_groups for p in group["params"]]
        places = [i for group in state_dict["param_groups"] for i in group["params"]]
        made = {}                                            # (all of it is read before anything of the optimizer's changes)
        for p, place in zip(params, places):
            saved = state_dict["state"].get(place)
            if not saved:
                continue
            fresh = made[p] = self._new_state(p)
            for key in self._keys():
                if not isinstance(saved.get(key), torch.Tensor) or saved[key].shape != fresh[key].shape:
                    raise ValueError("FusedAdamW: %s of parameter %d has shape %s, expected %s"
                                     % (key, place, getattr(saved.get(key), "shape", None), tuple(fresh[key].shape)))
                if fresh[key].dtype == torch.float8_e4m3fn and saved[key].dtype != torch.float8_e4m3fn:
                    raise ValueError("FusedAdamW: %s of parameter %d is %s, expected e4m3 values" % (key, place, saved[key].dtype))
                fresh[key].copy_(saved[key])
            if "step" not in saved:
                raise ValueError("FusedAdamW: parameter %d has no step count" % place)
            fresh["step"] = int(saved["step"])
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        self.seed = int(state_dict.get("seed", self.seed))
        self.state.update(made)


OPTIMIZERS = {
    "adam": partial(FusedAdam, amsgrad=True),
    "momentum": partial(FusedSGD, momentum=0.9, nesterov=True),
}
# Optimizers that the reference does not have.  Their weight decay is for the weights alone: make_optimizer gives them two groups.
DECOUPLED_OPTIMIZERS = {
    "adamw": FusedAdamW,
    "adamw8": partial(FusedAdamW, state_bits=8),
}


def decay_groups(named_parameters, weight_decay):
    """Parameter groups for a decoupled optimizer: matrices and convolution filters decay; biases, norms, PReLU slopes and the time
    constants of a state-space head (marked `no_decay`) do not."""
    decay, rest = [], []
    for _, p in named_parameters:
        (decay if p.dim() > 1 and not getattr(p, "no_decay", False) else rest).append(p)
    return [g for g in (dict(params=decay, weight_decay=weight_decay), dict(params=rest, weight_decay=0.0)) if g["params"]]


def make_optimizer(name, module, lr, weight_decay):
    """The optimizer `name` over a module's parameters: OPTIMIZERS as in the reference, DECOUPLED_OPTIMIZERS with their two groups."""
    if name in DECOUPLED_OPTIMIZERS:
        return DECOUPLED_OPTIMIZERS[name](decay_groups(module.named_parameters(), weight_decay), lr, weight_decay=weight_decay)
    return OPTIMIZERS[name](module.parameters(), lr, weight_decay=weight_decay)


class OneCycleScheduler:
    """Linear warm-up from min_lr to max_lr over the first 30 % of `max_steps`, then linear
    decay to min_lr / 1000 (reference ops/training.py:208-234).  `step()` sets the lr for the
    upcoming optimizer step."""

    def __init__(self, optimizer, min_lr, max_lr, max_steps):
        self.optimizer = optimizer
        self.min_lr = min_lr
        self.max_lr = max_lr
        self.max_steps = max_steps
        self.epoch = -1

    def lr_at(self, index):
        knee = int(round(self.max_steps * 0.3))
        if index < knee:
            return self.min_lr + (index / knee) * (self.max_lr - self.min_lr)
        frac = (index - knee) / (self.max_steps - knee)
        return self.max_lr + frac * (self.min_lr / 1e3 - self.max_lr)

    def step(self):
        self.epoch += 1
        lr = self.lr_at(self.epoch)
        for group in self.optimizer.param_groups:
            group["lr"] = lr


def make_scheduler(params, max_steps):
    """Descriptor -> callable(optimizer) building the scheduler (reference ops/training.py:15-34)."""
    name, *args = params.split("_")
    if name == "steplr":
        step_size, gamma = int(args[0]), float(args[1])
        return partial(StepLR, step_size=step_size, gamma=gamma)
    if name == "1cycle":
        min_lr, max_lr = float(args[0]), float(args[1])
        return partial(OneCycleScheduler, min_lr=min_lr, max_lr=max_lr, max_steps=max_steps)
    raise ValueError("unknown scheduler descriptor %r" % params)


def make_step(scheduler, epoch=None, step=None, val_score=None):
    """StepLR advances per epoch, 1cycle per training step (reference ops/training.py:37-43)."""
    if isinstance(scheduler, StepLR) and epoch is not None:
        scheduler.step(epoch)
    elif isinstance(scheduler, OneCycleScheduler) and step is not None:
        scheduler.step()


class CapturedTrainingStep:
    """One training step of a model -- forward, loss, backward, optimizer -- recorded ONCE as a HIP graph and replayed per batch.

    The same entry points with the same arguments in the same order as the eager step, so a replayed step equals the eager one
    (40 replays of one recording stay within 1.5e-5 of the eager logits over four steps, tools/dbg_graph.py); what it removes is
    the host: ~510 entry-point calls of Python per cfg-3 step.  On a host that issues the step faster than the GPU runs it
    (this one: 9.2 ms against 11.5 ms) that buys nothing -- bench.py keeps eager steps and offers `--graph`.

    What makes it legal: every entry point of libfsc_hip.so is capture-safe (include/fsc_hip.h: no allocation, no
    synchronisation, no host read-back); the step-dependent scalars of Adam travel through two device floats
    (fsc_adam_amsgrad_step_dev) refreshed in front of each replay; BatchNorm counters are bumped by a kernel.  What it needs:
    fixed batch shape, Adam or AdamW, accumulation_steps == 1, no dropout (its counter-based stream takes the offset by value), single
    GPU (no reducer), at least one eager step before (lazy state exists).  `model.training_step` semantics otherwise: returns
    (class_logits, per-sample loss, loss) -- static tensors, valid until the next call.

    Two rules for the caller, both enforced:
    * ONE NON-DEFAULT STREAM for everything -- the eager steps before, the recording, the replays: construct and call inside the
      same `with torch.cuda.stream(s):`.  With the eager steps on torch's default stream (the legacy null stream) and the graph
      on another, replays were wrong in ways that depended on where the host synchronised (NaN logits within three replays with
      a device synchronise after every step; a stalled loss, or a NaN in one run of six, with bench.py's pattern; correct with a
      read-back after every step) -- tools/dbg_graph5.py reproduces it; nothing in the library or in torch's strictest capture
      mode flags anything, and the same loop on one non-default stream is correct under every pattern tried.
    * NO tensor of an earlier step's autograd graph may be alive at the recording (drop the eager steps' logits / losses first):
      it keeps the parameters' AccumulateGrad nodes alive, which then run outside the recording.  The constructor drops the
      library's own references (the BatchNorm statistics stash), collects garbage, and refuses the recording if torch reports
      such a node.
    """

    def __init__(self, model, signal, labels):
        opt = model.optimizer
        if not isinstance(opt, (FusedAdam, FusedAdamW)):
            raise _lib.FscError("CapturedTrainingStep needs the fused Adam or AdamW optimizer")
        if model._reducer is not None or model.config.train.accumulation_steps != 1:
            raise _lib.FscError("CapturedTrainingStep: single GPU, accumulation_steps == 1")
        if float(model.config.network.output_dropout) > 0.0:
            raise _lib.FscError("CapturedTrainingStep: dropout draws from a host-side counter; capture needs output_dropout == 0")
        decoupled = isinstance(opt, FusedAdamW)
        trained = [p for group in opt.param_groups for p in group["params"] if p.requires_grad]
        if (len(opt.param_groups) != 1 and not decoupled) or not all(opt.state[p] for p in trained):
            raise _lib.FscError("CapturedTrainingStep: run one eager training step first (optimizer state must exist)")
        if decoupled and len({int(opt.state[p]["step"]) for p in trained}) != 1:
            raise _lib.FscError("CapturedTrainingStep: the parameters have taken different numbers of steps")
        stream = torch.cuda.current_stream(signal.device)
        if stream == torch.cuda.default_stream(signal.device):
            raise _lib.FscError("CapturedTrainingStep: run the training loop -- eager steps, this constructor, the replays -- inside "
                                "ONE `with torch.cuda.stream(s):` (not on the default stream; see the class docstring)")
        self.stream = stream
        self.model, self.opt = model, opt
        self.step_count = int(opt.state[trained[0]]["step"]) if trained else 0
        self.signal = signal.clone()
        self.labels = labels.clone()
        per_group = 4 if decoupled else 2
        self.factors = torch.zeros(per_group * len(opt.param_groups), device=signal.device, dtype=torch.float32)
        self._buf = (C.c_float * per_group)()
        self.graph = torch.cuda.CUDAGraph()
        opt.zero_grad()
        from .. import functional
        functional._PRESTATS.clear()             # (holds the last block output of the previous step, i.e. its autograd graph)
        gc.collect()
        opt.factors_dev = self.factors
        try:
            with warnings.catch_warnings(record=True) as caught:
                warnings.simplefilter("always")
                with torch.cuda.graph(self.graph, stream=stream, capture_error_mode=os.environ.get("FSC_CAPTURE_MODE", "relaxed")):
                    self.outputs = model.training_step(self.signal, self.labels)
        finally:
            opt.factors_dev = None
            # the recording ran the step's Python (not its kernels): undo the one host-side effect, the step counters of what got a gradient
            self._trained = [p for p in trained if int(opt.state[p]["step"]) != self.step_count]
            self.sync_state()
        self._places = self._where()
        stale = [w for w in caught if "AccumulateGrad" in str(w.message)]
        for w in caught:
            if w not in stale:
                warnings.warn_explicit(w.message, w.category, w.filename, w.lineno)
        if stale:
            self.graph = None
            raise _lib.FscError("CapturedTrainingStep: a tensor of an earlier step's autograd graph is still alive (its AccumulateGrad "
                                "nodes would run outside the recording); drop the previous steps' outputs before recording")

    def _tensors(self):
        """What the recorded optimizer step writes: parameters and moments as they are now."""
        return [t for p in self._trained for t in (p, *self.opt.state[p].values()) if isinstance(t, torch.Tensor) and t.is_cuda]

    def _where(self):
        return list(map(torch.Tensor.data_ptr, self._tensors()))

    def __call__(self, signal, labels):
        if self._where() != self._places:
            raise _lib.FscError("CapturedTrainingStep: parameters or moments are not where they were recorded (a checkpoint loaded or the model moved "
                                "since?); record the step again")
        if torch.cuda.current_stream(self.signal.device) != self.stream:
            raise _lib.FscError("CapturedTrainingStep: replay on the stream the step was recorded on")
        if tuple(signal.shape) != tuple(self.signal.shape) or tuple(labels.shape) != tuple(self.labels.shape):
            raise _lib.FscError("CapturedTrainingStep: recorded for a batch of shape %s / %s, got %s / %s (copy_ would broadcast)"
                                % (tuple(self.signal.shape), tuple(self.labels.shape), tuple(signal.shape), tuple(labels.shape)))
        self.signal.copy_(signal, non_blocking=True)
        self.labels.copy_(labels, non_blocking=True)
        self.step_count += 1
        # the replay rewrites parameters and BatchNorm buffers through raw pointers (no torch version bump by itself): the caches of an
        # inference forward between replays (packed fragments, folded eval-mode BatchNorm) must not survive it
        from .. import functional
        functional.forget_packed_weights()
        self.sync_state()                                 # (a checkpoint saved mid-run resumes with the right bias correction)
        to = self.factors.data_ptr()
        for group in self.opt.param_groups:
            b1, b2 = group["betas"]
            if isinstance(self.opt, FusedAdamW):
                _lib.load().fsc_adamw_step_factors(float(group["lr"]), b1, b2, float(group["weight_decay"]), self.step_count, self._buf)
            else:
                _lib.load().fsc_adam_step_factors(float(group["lr"]), b1, b2, self.step_count, self._buf)
            # (by-value kernel arguments: no host buffer that a later call could overwrite before an earlier copy has run)
            for value in self._buf:
                call("fsc_fill", to, float(value), 1, stream_ptr())
                to += 4
        self.graph.replay()
        if isinstance(self.opt, FusedAdamW):
            _mark_changed(self._tensors())
        return self.outputs

    def sync_state(self):
        """Write the step count back into the optimizer's state (state_dict compatibility) -- call before saving.  (Parameters that the recorded step
        does not change may have a state of earlier steps: it stays as it is.)"""
        for p in self._trained:
            self.opt.state[p]["step"] = self.step_count
