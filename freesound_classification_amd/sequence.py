"""Sequence operators of the state-space head: short causal convolution and selective scan, for whole sequences (with gradients)
and for single frames over a kept state.  Public through `functional` (`causal_conv`, `causal_conv_step`, `selective_scan`,
`selective_scan_step`, `ssm_head`).

Sequences are (N, T, D) with the channels last; tensors whose channels are contiguous are read in place whatever the strides of their other
axes (halves of one projection, time slices), others are copied first.  Activations are fp32, bf16 or fp16 (one type per call), parameters and
scan states fp32; sums and states are fp32 inside, with one rounding at each output.  `lengths` (N,) int32 marks padded batches: frames at and
behind lengths[n] are never read (they may hold anything), give zeros and get zero gradients, and states pass them by unchanged.  Infinities and NaN in
frames that exist go where the formulas take them and nowhere else.  First derivatives only, backwards only: others are refused.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import CausalConvArgs, ScanArgs, call, stream_ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_TAPS = 8
MAX_STATES = 64
_Tensor = torch.Tensor
_moved_on = torch.autograd.graph.increment_version           # (a graph that saved the state in front of the step must not use it)


def _fail(what, text, *args):
    raise _lib.FscError("%s: %s" % (what, text % args))


def _check(what, name, t, shape, dtype, device):
    """What is wrong with a tensor that is not a `dtype` tensor of `shape` on device number `device`."""
    if not isinstance(t, _Tensor):
        _fail(what, "%s must be a tensor, got %s", name, type(t).__name__)
    if not t.is_cuda:
        _fail(what, "%s: expected a device tensor, got %s (no CPU fallback)", name, t.device)
    if t.dtype != dtype:
        _fail(what, "%s is %s, expected %s", name, t.dtype, dtype)
    if tuple(t.shape) != tuple(shape):
        _fail(what, "%s has shape %s, expected %s", name, tuple(t.shape), tuple(shape))
    _fail(what, "%s is on %s, the current device is cuda:%d", name, t.device, device)


def _activation(what, name, t, shape, dtype, device):
    """One activation, checked, with contiguous channels."""
    if not (isinstance(t, _Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == device):
        _check(what, name, t, shape, dtype, device)
    strides = t.stride()
    if (strides[-1] != 1 and shape[-1] > 1) or (len(strides) > 2 and strides[1] > 1 << 26):      # (the kernels step over frames in 32 bits)
        t = t.clone(memory_format=torch.contiguous_format)       # (contiguous() keeps the strides of axes of length 1)
    return t


def _parameter(what, name, t, shape, device):
    """One fp32 tensor (parameter or state), checked, contiguous."""
    if not (isinstance(t, _Tensor) and t.dtype is torch.float32 and t.shape == shape and t.get_device() == device):
        _check(what, name, t, shape, torch.float32, device)
    return t if t.is_contiguous() else t.contiguous()


def _lengths(what, t, n, device):
    if t is None:
        return None
    if not (isinstance(t, _Tensor) and t.dtype is torch.int32 and t.shape == (n,) and t.get_device() == device):
        _check(what, "lengths", t, (n,), torch.int32, device)
    return t if t.is_contiguous() else t.contiguous()


def _state(what, name, t, shape, dtype, device):
    """A state that is updated in place: no copy may stand in for it."""
    if not (isinstance(t, _Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == device):
        _check(what, name, t, shape, dtype, device)
    if not t.is_contiguous():
        _fail(what, "%s is updated in place and must be contiguous", name)
    if t.requires_grad and torch.is_grad_enabled():
        _fail(what, "%s is updated in place and cannot require a gradient", name)
    return t


def _first(what, name, t, dims, shape):
    """The activation that sets the others' type and device."""
    if not isinstance(t, _Tensor) or t.dim() != dims:
        _fail(what, "%s must be a tensor (%s)", name, shape)
    device = t.get_device()
    if device < 0 or device != _lib._get_device():
        _check(what, name, t, t.shape, t.dtype, _lib._get_device() if t.is_cuda else -1)
    if t.dtype not in _DTYPES:
        _fail(what, "%s: fp32, bf16 or fp16, got %s", name, t.dtype)
    return _activation(what, name, t, t.shape, t.dtype, device), device


def _grad_needed(*tensors):
    return (torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in tensors])) or _has_tangent(tensors)


def _has_tangent(tensors):
    """Whether forward-mode derivatives arrive (they do not need requires_grad): autograd then refuses the function, which has none to pass on."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any([t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors])


def _one_frame(what, *tensors):
    if _grad_needed(*tensors):
        _fail(what, "a single frame has no gradient and no forward derivative: run it under torch.no_grad(), or the sequence operator for training")


def once(backward):
    """once_differentiable, whose own work (as much as a launch) is only done where a graph of the gradient is asked for."""
    guarded = once_differentiable(backward)
    return lambda ctx, *grads: (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)


def _addr(t):
    return 0 if t is None else t.data_ptr()


def _room(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


# ------------------------------------------------------------------------------ causal convolution
def _conv_args(x, weight, bias, silu, lengths, initial, y=None, final=None, dy=None, dfinal=None, dx=None, di=None, dw=None, db=None, ws=None):
    (n, t, d), (xb, xt, _) = x.shape, x.stride()
    gb, gt = (0, 0) if dy is None else dy.stride()[:2]
    return CausalConvArgs.packed(n, t, d, weight.shape[1], _DTYPES[x.dtype], silu, x.data_ptr(), xb, xt, weight.data_ptr(), _addr(bias), _addr(lengths),
                                 _addr(initial), _addr(y), _addr(final), _addr(dy), gb, gt, _addr(dfinal), _addr(dx), _addr(di), _addr(dw),
                                 _addr(db), _addr(ws))


def _conv_forward(x, weight, bias, initial, lengths, silu, want_final):
    y = x.new_empty(x.shape)
    final = x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2])) if want_final else None
    call("fsc_causal_conv_fwd", _conv_args(x, weight, bias, silu, lengths, initial, y, final), stream_ptr())
    return y, final


class CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial, lengths, silu, want_final):
        ctx.save_for_backward(x, weight, bias, initial, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return _conv_forward(x, weight, bias, initial, lengths, silu, want_final)

    @staticmethod
    @once
    def backward(ctx, dy, dfinal):
        if dy is None and dfinal is None:
            return (None,) * 7
        x, weight, bias, initial, lengths = ctx.saved_tensors
        if dy is not None:
            dy = _activation("causal_conv", "the gradient", dy, x.shape, x.dtype, x.get_device())
        dfinal = None if dfinal is None else dfinal.contiguous()
        dx, dw = x.new_empty(x.shape), weight.new_empty(weight.shape)
        db = None if bias is None else bias.new_empty(bias.shape)
        di = None if initial is None else initial.new_empty(initial.shape)
        same = (x, weight, bias, ctx.silu, lengths, initial, None, None, dy, dfinal, dx, di, dw, db)
        ws = _room(_lib.load().fsc_causal_conv_bwd_workspace_bytes(_conv_args(*same)), x)
        call("fsc_causal_conv_bwd", _conv_args(*same, ws), stream_ptr())
        return dx, dw, db, di, None, None, None


def _conv_inputs(what, x, dims, weight, bias, activation):
    x, device = _first(what, "x", x, dims, "batch, frames, channels" if dims == 3 else "batch, channels")
    if activation not in ("silu", None):
        _fail(what, "activation must be 'silu' or None, got %r", activation)
    if not isinstance(weight, _Tensor) or weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_TAPS:
        _fail(what, "weight must be (channels, taps) with 1 to %d taps", MAX_TAPS)
    d = x.shape[-1]
    weight = _parameter(what, "weight", weight, (d, weight.shape[1]), device)
    bias = None if bias is None else _parameter(what, "bias", bias, (d,), device)
    return x, weight, bias, device


def causal_conv(x, weight, bias=None, activation="silu", lengths=None, initial=None, return_final=False):
    """y[n, t, c] = act(bias[c] + sum_k weight[c, k] xin[n, t + k, c]) with xin = the K - 1 frames `initial` (N, K - 1, D; zeros without
    it) followed by x (N, T, D); weight (D, K), K <= 8; act = SiLU or, with activation=None, nothing.  Returns y, or (y, final) with
    final (N, K - 1, D) the last frames of each sequence: `initial` of what follows, and the window of causal_conv_step.  Differentiable in x,
    weight, bias and initial, through y and final."""
    what = "causal_conv"
    x, weight, bias, device = _conv_inputs(what, x, 3, weight, bias, activation)
    n, _, d = x.shape
    if initial is not None:
        initial = _activation(what, "initial", initial, (n, weight.shape[1] - 1, d), x.dtype, device).contiguous()
    args = x, weight, bias, initial, _lengths(what, lengths, n, device), int(activation is not None), return_final
    y, final = CausalConvFn.apply(*args) if _grad_needed(x, weight, bias, initial) else _conv_forward(*args)
    return (y, final) if return_final else y


def causal_conv_step(x, window, weight, bias=None, activation="silu"):
    """One frame x (N, D) behind the K - 1 frames of `window` (N, K - 1, D), which moves on by one frame IN PLACE.  Returns y (N, D)."""
    what = "causal_conv_step"
    x, weight, bias, device = _conv_inputs(what, x, 2, weight, bias, activation)
    n, d = x.shape
    taps = weight.shape[1]
    window = _state(what, "window", window, (n, taps - 1, d), x.dtype, device)
    _one_frame(what, x, weight, bias, window)
    y = x.new_empty((n, d))
    call("fsc_causal_conv_step",
         CausalConvArgs.packed(n, 1, d, taps, _DTYPES[x.dtype], int(activation is not None), x.data_ptr(), x.stride(0), 0, weight.data_ptr(),
                               _addr(bias), 0, window.data_ptr(), y.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0), stream_ptr())
    _moved_on(window)
    return y


# ------------------------------------------------------------------------------ selective scan
def _scan_args(u, dt, a_log, b, c, d, z, dt_bias, soft, lengths, initial, y=None, final=None, kept=None, ws=None, dy=None, dfinal=None, grads=(0,) * 9):
    """u, dt, z (N, T, D) and b, c (N, T, G, S), or without T: a single frame."""
    if u.dim() == 3:
        n, t, channels = u.shape
        (ub, ut, _), (tb, tt, _), (bb, bt, bg, _), (cb, ct, cg, _) = u.stride(), dt.stride(), b.stride(), c.stride()
        zb, zt = (0, 0) if z is None else z.stride()[:2]
    else:
        (n, channels), t = u.shape, 1
        (ub, _), (tb, _), (bb, bg, _), (cb, cg, _) = u.stride(), dt.stride(), b.stride(), c.stride()
        zb, ut, tt, bt, ct, zt = 0 if z is None else z.stride(0), 0, 0, 0, 0, 0
    gb, gt = (0, 0) if dy is None else dy.stride()[:2]
    return ScanArgs.packed(n, t, channels, a_log.shape[1], b.shape[-2], _DTYPES[u.dtype], soft, u.data_ptr(), dt.data_ptr(), _addr(z), b.data_ptr(),
                           c.data_ptr(), ub, ut, tb, tt, zb, zt, bb, bt, bg, cb, ct, cg, a_log.data_ptr(), _addr(d), _addr(dt_bias), _addr(lengths),
                           _addr(initial), _addr(y), _addr(final), _addr(kept), _addr(ws), _addr(dy), gb, gt, _addr(dfinal), *grads)


def _scan_forward(u, dt, a_log, b, c, d, z, dt_bias, initial, lengths, soft, want_final, keep=False):
    lib = _lib.load()
    y = u.new_empty(u.shape)
    final = a_log.new_empty((u.shape[0],) + tuple(a_log.shape)) if want_final else None
    same = (u, dt, a_log, b, c, d, z, dt_bias, soft, lengths, initial, y, final)
    plan = _scan_args(*same)
    kept = _room(lib.fsc_selective_scan_checkpoint_bytes(plan), u) if keep else None
    nbytes = lib.fsc_selective_scan_workspace_bytes(plan, 0)
    ws = _room(nbytes, u)
    call("fsc_selective_scan_fwd", _scan_args(*same, kept, ws) if keep or nbytes else plan, stream_ptr())
    return y, final, kept


class SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, dt, a_log, b, c, d, z, dt_bias, initial, lengths, soft, want_final):
        y, final, kept = _scan_forward(u, dt, a_log, b, c, d, z, dt_bias, initial, lengths, soft, want_final, keep=True)
        ctx.save_for_backward(u, dt, a_log, b, c, d, z, dt_bias, initial, lengths, kept)
        ctx.soft = soft
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @once
    def backward(ctx, dy, dfinal):
        if dy is None and dfinal is None:
            return (None,) * 12
        u, dt, a_log, b, c, d, z, dt_bias, initial, lengths, kept = ctx.saved_tensors
        if dy is not None:
            dy = _activation("selective_scan", "the gradient", dy, u.shape, u.dtype, u.get_device())
        dfinal = None if dfinal is None else dfinal.contiguous()
        made = [None if t is None else t.new_empty(t.shape) for t in (u, dt, z, b, c, a_log, d, dt_bias, initial)]
        same = (u, dt, a_log, b, c, d, z, dt_bias, ctx.soft, lengths, initial, None, None, kept)
        ws = _room(_lib.load().fsc_selective_scan_workspace_bytes(_scan_args(*same), 1), u)
        call("fsc_selective_scan_bwd", _scan_args(*same, ws, dy, dfinal, [_addr(t) for t in made]), stream_ptr())
        du, ddt, dz, db, dc, da, dd, dbias, di = made
        return du, ddt, da, db, dc, dd, dz, dbias, di, None, None, None


def _scan_inputs(what, dims, u, dt, a_log, b, c, d, z, dt_bias):
    """Checks what the sequence (dims = 3) and the single-frame form (2) share; B and C come back with a groups axis."""
    u, device = _first(what, "u", u, dims, "batch, frames, channels" if dims == 3 else "batch, channels")
    shape, dtype = u.shape, u.dtype
    lead, channels = shape[:-1], shape[-1]
    if not isinstance(a_log, _Tensor) or a_log.dim() != 2 or not 1 <= a_log.shape[1] <= MAX_STATES:
        _fail(what, "a_log must be (channels, states) with 1 to %d states", MAX_STATES)
    states = a_log.shape[1]
    a_log = _parameter(what, "a_log", a_log, (channels, states), device)
    dt = _activation(what, "dt", dt, shape, dtype, device)
    z = None if z is None else _activation(what, "z", z, shape, dtype, device)
    rows = []
    for name, t in (("b", b), ("c", c)):
        if isinstance(t, _Tensor) and t.dim() == dims:
            t = t.unsqueeze(-2)
        if not isinstance(t, _Tensor) or t.dim() != dims + 1 or t.shape[-2] < 1 or channels % t.shape[-2]:
            _fail(what, "%s must be (%s, [groups,] states) with groups dividing the %d channels", name, "batch, frames" if dims == 3 else "batch", channels)
        rows.append(_activation(what, name, t, lead + (t.shape[-2], states), dtype, device))
    b, c = rows
    if b.shape != c.shape:
        _fail(what, "b has %d groups, c %d", b.shape[-2], c.shape[-2])
    d = None if d is None else _parameter(what, "d", d, (channels,), device)
    dt_bias = None if dt_bias is None else _parameter(what, "dt_bias", dt_bias, (channels,), device)
    return u, dt, a_log, b, c, d, z, dt_bias, device


def selective_scan(u, dt, a_log, b, c, d=None, z=None, dt_bias=None, softplus=True, lengths=None, initial=None, return_final=False):
    """h_t = exp(delta_t A) h_{t-1} + delta_t u_t B_t, y_t = (C_t . h_t + d u_t) silu(z_t) with delta = softplus(dt + dt_bias)
    (softplus=False: dt + dt_bias) and A = -exp(a_log).  u, dt, z (N, T, D); a_log (D, S), S <= 64; b, c (N, T, S) or (N, T, G, S):
    channel j belongs to group j // (D / G); d, dt_bias (D,); initial (N, D, S) fp32 or None (zeros).  Returns y (N, T, D), or
    (y, final) with the state behind each sequence's last frame.  Differentiable in every tensor but lengths, through y and final."""
    what = "selective_scan"
    u, dt, a_log, b, c, d, z, dt_bias, device = _scan_inputs(what, 3, u, dt, a_log, b, c, d, z, dt_bias)
    n = u.shape[0]
    if initial is not None:
        initial = _parameter(what, "initial", initial, (n,) + tuple(a_log.shape), device)
    args = u, dt, a_log, b, c, d, z, dt_bias, initial, _lengths(what, lengths, n, device), int(bool(softplus)), return_final
    if _grad_needed(u, dt, a_log, b, c, d, z, dt_bias, initial):
        y, final = SelectiveScanFn.apply(*args)
    else:
        y, final, _ = _scan_forward(*args)
    return (y, final) if return_final else y


def selective_scan_step(u, dt, a_log, b, c, state, d=None, z=None, dt_bias=None, softplus=True):
    """One frame: u, dt, z (N, D), b, c (N, S) or (N, G, S); `state` (N, D, S) fp32 moves on by one frame IN PLACE.  Returns y (N, D)."""
    what = "selective_scan_step"
    u, dt, a_log, b, c, d, z, dt_bias, device = _scan_inputs(what, 2, u, dt, a_log, b, c, d, z, dt_bias)
    state = _state(what, "state", state, (u.shape[0],) + tuple(a_log.shape), torch.float32, device)
    _one_frame(what, u, dt, a_log, b, c, d, z, dt_bias, state)
    y = u.new_empty(u.shape)
    call("fsc_selective_scan_step", _scan_args(u, dt, a_log, b, c, d, z, dt_bias, int(bool(softplus)), None, None, y, state), stream_ptr())
    _moved_on(state)
    return y
