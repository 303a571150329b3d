"""Sequence operators of the state-space head: short causal convolution and selective scan, for whole sequences (with gradients)
and for single frames over a kept state.  Public through `functional` (`causal_conv`, `causal_conv_step`, `selective_scan`,
`selective_scan_step`, `ssm_head`).

Sequences are (N, T, D) with the channels last; tensors whose channels are contiguous are read in place whatever the strides of their other
axes (halves of one projection, time slices), others are copied first.  Activations are fp32, bf16 or fp16 (one type per call), parameters and
scan states fp32; sums and states are fp32 inside, with one rounding at each output.  `lengths` (N,) int32 marks padded batches: frames at and
behind lengths[n] are never read (they may hold anything), give zeros and get zero gradients, and states pass them by unchanged.
"""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import CausalConvArgs, ScanArgs, call, ptr, stream_ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_TAPS = 8
MAX_STATES = 64


def _fail(what, text, *args):
    raise _lib.FscError("%s: %s" % (what, text % args))


def _activation(what, name, t, shape, dtype=None):
    """Checks one activation and returns it with contiguous channels."""
    if not isinstance(t, torch.Tensor):
        _fail(what, "%s must be a tensor, got %s", name, type(t).__name__)
    if not t.is_cuda:
        _fail(what, "%s: expected a device tensor, got %s (no CPU fallback)", name, t.device)
    if t.dtype not in _DTYPES:
        _fail(what, "%s: fp32, bf16 or fp16, got %s", name, t.dtype)
    if dtype is not None and t.dtype != dtype:
        _fail(what, "%s is %s, the other activations %s", name, t.dtype, dtype)
    if tuple(t.shape) != tuple(shape):
        _fail(what, "%s has shape %s, expected %s", name, tuple(t.shape), tuple(shape))
    _same_device(what, name, t)
    if (t.shape[-1] > 1 and t.stride(-1) != 1) or (t.dim() > 2 and t.stride(1) > 1 << 26):      # (the kernels step over frames in 32 bits)
        t = t.contiguous()
    return t


def _same_device(what, name, t):
    if t.device.index != _lib._get_device():
        _fail(what, "%s is on %s, the current device is cuda:%d", name, t.device, torch.cuda.current_device())


def _parameter(what, name, t, shape, optional=False):
    """Checks one fp32 tensor (parameter or state) and returns it contiguous."""
    if t is None and optional:
        return None
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32:
        _fail(what, "%s must be an fp32 device tensor", name)
    if tuple(t.shape) != tuple(shape):
        _fail(what, "%s has shape %s, expected %s", name, tuple(t.shape), tuple(shape))
    _same_device(what, name, t)
    return t.contiguous()


def _lengths(what, t, n):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int32 or tuple(t.shape) != (n,):
        _fail(what, "lengths must be an int32 device tensor of shape (%d,)", n)
    _same_device(what, "lengths", t)
    return t.contiguous()


def _state(what, name, t, shape, dtype):
    """A state that is updated in place: no copy may stand in for it."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        _fail(what, "%s must be a contiguous %s device tensor of shape %s", name, dtype, tuple(shape))
    if t.requires_grad and torch.is_grad_enabled():
        _fail(what, "%s is updated in place and cannot require a gradient", name)
    _same_device(what, name, t)
    return t


def _no_grad_needed(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        _fail(what, "a single frame has no gradient: run it under torch.no_grad(), or the sequence operator for training")


def _addr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, like):
    return torch.empty(max(1, nbytes), device=like.device, dtype=torch.uint8) if nbytes else None


# ------------------------------------------------------------------------------ causal convolution
def _conv_args(x, weight, bias, silu, lengths, initial):
    n, t, d = x.shape
    return CausalConvArgs(batch=n, length=t, channels=d, taps=weight.shape[1], dtype=_DTYPES[x.dtype], silu=int(silu), x=x.data_ptr(),
                          x_batch=x.stride(0), x_time=x.stride(1), weight=weight.data_ptr(), bias=_addr(bias), lengths=_addr(lengths),
                          initial=_addr(initial))


class CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial, lengths, silu, want_final):
        n, t, d = x.shape
        args = _conv_args(x, weight, bias, silu, lengths, initial)
        y = torch.empty((n, t, d), device=x.device, dtype=x.dtype)
        final = torch.empty((n, weight.shape[1] - 1, d), device=x.device, dtype=x.dtype) if want_final else None
        args.y, args.final = y.data_ptr(), _addr(final)
        call("fsc_causal_conv_fwd", C.byref(args), stream_ptr())
        ctx.save_for_backward(x, weight, bias, initial, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, weight, bias, initial, lengths = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 7
        args = _conv_args(x, weight, bias, ctx.silu, lengths, initial)
        if dy is not None:
            dy = _activation("causal_conv", "the gradient", dy, x.shape, x.dtype)
            args.dy, args.dy_batch, args.dy_time = dy.data_ptr(), dy.stride(0), dy.stride(1)
        dfinal = None if dfinal is None else dfinal.contiguous()
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        dw = torch.empty_like(weight)
        db = None if bias is None else torch.empty_like(bias)
        di = None if initial is None else torch.empty_like(initial)
        ws = _workspace(_lib.load().fsc_causal_conv_bwd_workspace_bytes(C.byref(args)), x)
        args.dfinal, args.dx, args.dinitial = _addr(dfinal), dx.data_ptr(), _addr(di)
        args.dweight, args.dbias, args.workspace = dw.data_ptr(), _addr(db), _addr(ws)
        call("fsc_causal_conv_bwd", C.byref(args), stream_ptr())
        return dx, dw, db, di, None, None, None


def _silu_flag(what, activation):
    if activation not in ("silu", None):
        _fail(what, "activation must be 'silu' or None, got %r", activation)
    return activation == "silu"


def _conv_parameters(what, d, weight, bias):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_TAPS:
        _fail(what, "weight must be (channels, taps) with 1 to %d taps", MAX_TAPS)
    return _parameter(what, "weight", weight, (d, weight.shape[1])), _parameter(what, "bias", bias, (d,), optional=True)


def causal_conv(x, weight, bias=None, activation="silu", lengths=None, initial=None, return_final=False):
    """y[n, t, c] = act(bias[c] + sum_k weight[c, k] xin[n, t + k, c]) with xin = the K - 1 frames `initial` (N, K - 1, D; zeros without
    it) followed by x (N, T, D); weight (D, K), K <= 8; act = SiLU or, with activation=None, nothing.  Returns y, or (y, final) with
    final (N, K - 1, D) the last frames of each sequence: `initial` of what follows, and the window of causal_conv_step.  Differentiable in x,
    weight, bias and initial, through y and final."""
    what = "causal_conv"
    silu = _silu_flag(what, activation)
    if not isinstance(x, torch.Tensor) or x.dim() != 3:
        _fail(what, "x must be (batch, frames, channels)")
    x = _activation(what, "x", x, x.shape)
    n, _, d = x.shape
    weight, bias = _conv_parameters(what, d, weight, bias)
    if initial is not None:
        initial = _activation(what, "initial", initial, (n, weight.shape[1] - 1, d), x.dtype).contiguous()
    y, final = CausalConvFn.apply(x, weight, bias, initial, _lengths(what, lengths, n), silu, return_final)
    return (y, final) if return_final else y


def causal_conv_step(x, window, weight, bias=None, activation="silu"):
    """One frame x (N, D) behind the K - 1 frames of `window` (N, K - 1, D), which moves on by one frame IN PLACE.  Returns y (N, D)."""
    what = "causal_conv_step"
    silu = _silu_flag(what, activation)
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        _fail(what, "x must be (batch, channels)")
    x = _activation(what, "x", x, x.shape)
    n, d = x.shape
    weight, bias = _conv_parameters(what, d, weight, bias)
    window = _state(what, "window", window, (n, weight.shape[1] - 1, d), x.dtype)
    _no_grad_needed(what, x, weight, bias)
    y = torch.empty((n, d), device=x.device, dtype=x.dtype)
    args = _conv_args(x.unsqueeze(1), weight, bias, silu, None, window)
    args.y = y.data_ptr()
    call("fsc_causal_conv_step", C.byref(args), stream_ptr())
    return y


# ------------------------------------------------------------------------------ selective scan
def _scan_args(u, dt, a_log, b, c, d, z, dt_bias, softplus, lengths, initial):
    n, t, channels = u.shape
    args = ScanArgs(batch=n, length=t, channels=channels, states=b.shape[3], groups=b.shape[2], dtype=_DTYPES[u.dtype],
                    softplus=int(softplus), u=u.data_ptr(), u_batch=u.stride(0), u_time=u.stride(1), dt=dt.data_ptr(),
                    dt_batch=dt.stride(0), dt_time=dt.stride(1), b=b.data_ptr(), b_batch=b.stride(0), b_time=b.stride(1),
                    b_group=b.stride(2), c=c.data_ptr(), c_batch=c.stride(0), c_time=c.stride(1), c_group=c.stride(2),
                    a_log=a_log.data_ptr(), d=_addr(d), dt_bias=_addr(dt_bias), lengths=_addr(lengths), initial=_addr(initial))
    if z is not None:
        args.z, args.z_batch, args.z_time = z.data_ptr(), z.stride(0), z.stride(1)
    return args


class SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, dt, a_log, b, c, d, z, dt_bias, initial, lengths, softplus, want_final):
        lib = _lib.load()
        args = _scan_args(u, dt, a_log, b, c, d, z, dt_bias, softplus, lengths, initial)
        y = torch.empty(u.shape, device=u.device, dtype=u.dtype)
        final = torch.empty((u.shape[0],) + tuple(a_log.shape), device=u.device, dtype=torch.float32) if want_final else None
        kept = None
        if any(ctx.needs_input_grad):
            kept = _workspace(lib.fsc_selective_scan_checkpoint_bytes(C.byref(args)), u)
        ws = _workspace(lib.fsc_selective_scan_workspace_bytes(C.byref(args), 0), u)
        args.y, args.final, args.checkpoints, args.workspace = y.data_ptr(), _addr(final), _addr(kept), _addr(ws)
        call("fsc_selective_scan_fwd", C.byref(args), stream_ptr())
        ctx.save_for_backward(u, dt, a_log, b, c, d, z, dt_bias, initial, lengths)
        ctx.kept, ctx.softplus = kept, softplus
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        u, dt, a_log, b, c, d, z, dt_bias, initial, lengths = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 12
        args = _scan_args(u, dt, a_log, b, c, d, z, dt_bias, ctx.softplus, lengths, initial)
        if dy is not None:
            dy = _activation("selective_scan", "the gradient", dy, u.shape, u.dtype)
            args.dy, args.dy_batch, args.dy_time = dy.data_ptr(), dy.stride(0), dy.stride(1)
        dfinal = None if dfinal is None else dfinal.contiguous()

        def like(t):
            return None if t is None else torch.empty(t.shape, device=t.device, dtype=t.dtype)

        du, ddt, dz, db, dc = like(u), like(dt), like(z), like(b), like(c)
        da, dd, dbias, di = like(a_log), like(d), like(dt_bias), like(initial)
        ws = _workspace(_lib.load().fsc_selective_scan_workspace_bytes(C.byref(args), 1), u)
        args.checkpoints, args.workspace, args.dfinal = _addr(ctx.kept), _addr(ws), _addr(dfinal)
        args.du, args.ddt, args.dz, args.db, args.dc = du.data_ptr(), ddt.data_ptr(), _addr(dz), db.data_ptr(), dc.data_ptr()
        args.da_log, args.dd, args.ddt_bias, args.dinitial = da.data_ptr(), _addr(dd), _addr(dbias), _addr(di)
        call("fsc_selective_scan_bwd", C.byref(args), stream_ptr())
        return du, ddt, da, db, dc, dd, dz, dbias, di, None, None, None


def _scan_inputs(what, frames, u, dt, a_log, b, c, d, z, dt_bias):
    """Checks what the sequence and the single-frame form share; B and C come back with a groups axis."""
    dims = 3 if frames else 2
    if not isinstance(u, torch.Tensor) or u.dim() != dims:
        _fail(what, "u must be (batch, %schannels)", "frames, " if frames else "")
    u = _activation(what, "u", u, u.shape)
    lead, channels = tuple(u.shape[:-1]), u.shape[-1]
    if not isinstance(a_log, torch.Tensor) or a_log.dim() != 2 or not 1 <= a_log.shape[1] <= MAX_STATES:
        _fail(what, "a_log must be (channels, states) with 1 to %d states", MAX_STATES)
    states = a_log.shape[1]
    a_log = _parameter(what, "a_log", a_log, (channels, states))
    dt = _activation(what, "dt", dt, u.shape, u.dtype)
    z = None if z is None else _activation(what, "z", z, u.shape, u.dtype)

    def rows(name, t):
        if isinstance(t, torch.Tensor) and t.dim() == dims:
            t = t.unsqueeze(-2)
        if not isinstance(t, torch.Tensor) or t.dim() != dims + 1 or t.shape[-2] < 1 or channels % t.shape[-2]:
            _fail(what, "%s must be %s[groups, ] states), groups dividing the %d channels", name, "(batch, frames, " if frames else "(batch, ", channels)
        return _activation(what, name, t, lead + (t.shape[-2], states), u.dtype)

    b, c = rows("b", b), rows("c", c)
    if b.shape != c.shape:
        _fail(what, "b has %d groups, c %d", b.shape[-2], c.shape[-2])
    return u, dt, a_log, b, c, _parameter(what, "d", d, (channels,), True), z, _parameter(what, "dt_bias", dt_bias, (channels,), True)


def selective_scan(u, dt, a_log, b, c, d=None, z=None, dt_bias=None, softplus=True, lengths=None, initial=None, return_final=False):
    """h_t = exp(delta_t A) h_{t-1} + delta_t u_t B_t, y_t = (C_t . h_t + d u_t) silu(z_t) with delta = softplus(dt + dt_bias)
    (softplus=False: dt + dt_bias) and A = -exp(a_log).  u, dt, z (N, T, D); a_log (D, S), S <= 64; b, c (N, T, S) or (N, T, G, S):
    channel j belongs to group j // (D / G); d, dt_bias (D,); initial (N, D, S) fp32 or None (zeros).  Returns y (N, T, D), or
    (y, final) with the state behind each sequence's last frame.  Differentiable in every tensor but lengths, through y and final."""
    what = "selective_scan"
    u, dt, a_log, b, c, d, z, dt_bias = _scan_inputs(what, True, u, dt, a_log, b, c, d, z, dt_bias)
    n = u.shape[0]
    initial = _parameter(what, "initial", initial, (n,) + tuple(a_log.shape), optional=True)
    y, final = SelectiveScanFn.apply(u, dt, a_log, b, c, d, z, dt_bias, initial, _lengths(what, lengths, n), bool(softplus), return_final)
    return (y, final) if return_final else y


def selective_scan_step(u, dt, a_log, b, c, state, d=None, z=None, dt_bias=None, softplus=True):
    """One frame: u, dt, z (N, D), b, c (N, S) or (N, G, S); `state` (N, D, S) fp32 moves on by one frame IN PLACE.  Returns y (N, D)."""
    what = "selective_scan_step"
    u, dt, a_log, b, c, d, z, dt_bias = _scan_inputs(what, False, u, dt, a_log, b, c, d, z, dt_bias)
    state = _state(what, "state", state, (u.shape[0],) + tuple(a_log.shape), torch.float32)
    _no_grad_needed(what, u, dt, a_log, b, c, d, z, dt_bias)
    one = lambda t: None if t is None else t.unsqueeze(1)  # noqa: E731
    y = torch.empty(u.shape, device=u.device, dtype=u.dtype)
    args = _scan_args(one(u), one(dt), a_log, one(b), one(c), d, one(z), dt_bias, softplus, None, None)
    args.y, args.final = y.data_ptr(), state.data_ptr()
    call("fsc_selective_scan_step", C.byref(args), stream_ptr())
    return y
