"""Plain 64-bit recurrences of the state-space head's operators and of the decoupled optimizer: one frame after the other, one formula a
line, differentiable by autograd.  Test infrastructure."""
import numpy as np
import torch


def causal_conv(x, weight, bias=None, silu=True, lengths=None, initial=None):
    """x (N, T, D), weight (D, K) -> (y, final)."""
    n, t, d = x.shape
    k = weight.shape[1]
    ends = [t] * n if lengths is None else [min(max(int(v), 0), t) for v in lengths]
    before = torch.zeros(n, k - 1, d, dtype=x.dtype) if initial is None else initial
    y, final = [], []
    for i in range(n):
        rows = torch.cat([before[i], x[i, :ends[i]]])
        pre = torch.zeros(ends[i], d, dtype=x.dtype) if bias is None else bias.expand(ends[i], d)
        for j in range(k):
            pre = pre + rows[j:j + ends[i]] * weight[:, j]
        out = pre * torch.sigmoid(pre) if silu else pre
        y.append(torch.cat([out, torch.zeros(t - ends[i], d, dtype=x.dtype)]))
        final.append(rows[ends[i]:])
    return torch.stack(y), torch.stack(final)


def selective_scan(u, dt, a_log, b, c, d=None, z=None, dt_bias=None, softplus=True, lengths=None, initial=None):
    """u, dt, z (N, T, D), a_log (D, S), b, c (N, T, G, S) -> (y, final)."""
    n, t, channels = u.shape
    groups, states = b.shape[2:]
    ends = [t] * n if lengths is None else [min(max(int(v), 0), t) for v in lengths]
    rate = -torch.exp(a_log)
    y, final = [], []
    for i in range(n):
        h = torch.zeros(channels, states, dtype=u.dtype) if initial is None else initial[i]
        rows = []
        for k in range(ends[i]):
            raw = dt[i, k] if dt_bias is None else dt[i, k] + dt_bias
            delta = torch.nn.functional.softplus(raw, threshold=50) if softplus else raw
            bk, ck = (v[i, k].repeat_interleave(channels // groups, 0) for v in (b, c))
            h = torch.exp(delta[:, None] * rate) * h + (delta * u[i, k])[:, None] * bk
            out = (h * ck).sum(1)
            if d is not None:
                out = out + d * u[i, k]
            if z is not None:
                out = out * z[i, k] * torch.sigmoid(z[i, k])
            rows.append(out)
        rows += [torch.zeros(channels, dtype=u.dtype)] * (t - ends[i])
        y.append(torch.stack(rows) if rows else torch.zeros(0, channels, dtype=u.dtype))
        final.append(h)
    return torch.stack(y), torch.stack(final)


def ssm_head(out, p, inner, rank, states, eps=1e-5):
    """The aggregation head on a block output (N, C, H, W); p: its parameters by name."""
    x = out.mean(2).permute(0, 2, 1)
    x = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + eps) * p["norm.weight"] + p["norm.bias"]
    xz = x @ p["in_proj.weight"].t() + p["in_proj.bias"]
    x, z = xz[..., :inner], xz[..., inner:]
    x, _ = causal_conv(x, p["conv_weight"], p["conv_bias"])
    proj = x @ p["x_proj.weight"].t()
    dt = proj[..., :rank] @ p["dt_proj.weight"].t()
    b, c = proj[..., rank:rank + states].unsqueeze(2), proj[..., rank + states:].unsqueeze(2)
    y, _ = selective_scan(x, dt, p["a_log"], b, c, p["d"], z, p["dt_proj.bias"])
    return y.mean(1)


# ---------------------------------------------------------------------------------------------------------------- AdamW
def adamw(p, g, m, v, step, lr, beta1, beta2, eps, weight_decay):
    """One step in the precision of its inputs; returns (p, m, v)."""
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    p = p * (1 - lr * weight_decay) - lr / (1 - beta1 ** step) * m / (np.sqrt(v) / np.sqrt(1 - beta2 ** step) + eps)
    return p, m, v


_F = np.float32


def _mix(x):
    x = np.asarray(x, dtype=np.uint64)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x9E3779B9)) & np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0xB7E15163)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def random_bits(salt, step, count):
    key = _mix((_mix(salt & 0xFFFFFFFF) + np.uint64(step & 0xFFFFFF)) & np.uint64(0xFFFFFFFF))
    return _mix(np.arange(count, dtype=np.uint64) ^ key).astype(np.uint32)


def e4m3_value(code):
    """The value of each 8-bit pattern: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7F / 0xFF not a number."""
    code = np.asarray(code, dtype=np.int64)
    e, m = (code >> 3) & 15, code & 7
    value = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    value = np.where((code & 0x7F) == 0x7F, np.nan, value)
    return np.where(code & 0x80, -value, value).astype(_F)


def held8(x, bits16, keep_positive):
    """(patterns, scales): e4m3 values of blocks of 256 over a scale, rounded by 16 random bits; x is fp32 and every operation rounds to it."""
    count = x.size
    rows = np.pad(x, (0, -count % 256)).reshape(-1, 256)
    top = np.where(np.isfinite(rows), np.abs(rows), _F(0)).max(1)
    scale = top * (_F(1) / _F(448))
    dead = scale < np.finfo(_F).tiny
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inverse = np.where(dead, _F(0), (_F(1) / top) * _F(448))
        y = (rows * inverse[:, None]).reshape(-1)[:count]
    size = np.abs(y)
    pattern = size.view(np.uint32).astype(np.int64)
    bits16 = bits16.astype(np.int64)
    normal = ((pattern + (bits16 << 4)) >> 20) - (120 << 3)
    with np.errstate(invalid="ignore"):
        small = np.floor(np.where(np.isfinite(size), size, 0) * _F(512) + bits16.astype(_F) * _F(2.0 ** -16)).astype(np.int64)
    code = np.minimum(np.where(size >= _F(2.0 ** -6), normal, small), 0x7E)
    if keep_positive:
        code = np.where((code == 0) & (y > 0), 1, code)
    code = np.where(np.isfinite(y), code | np.where(np.signbit(y), 0x80, 0), 0x7F)
    return code.astype(np.uint8), np.where(dead, _F(0), scale)


def adamw8(p, g, codes, scales, salt, step, lr, beta1, beta2, eps, weight_decay):
    """One step with held moments, every operation rounded to fp32.  codes / scales: (m, r).  Returns (p fp32, codes, scales)."""
    count = p.size
    m, r = (e4m3_value(codes[i]) * np.repeat(scales[i], 256)[:count] for i in (0, 1))
    p, g = p.astype(_F), g.astype(_F)
    m = m * _F(beta1) + g * _F(1 - beta1)
    v = (r * r) * _F(beta2) + (g * g) * _F(1 - beta2)
    r = np.sqrt(v)
    root, size = _F(1 / np.sqrt(1 - beta2 ** step)), _F(lr / (1 - beta1 ** step))
    with np.errstate(divide="ignore", invalid="ignore"):
        p = p * _F(1 - lr * weight_decay) - (m / (r * root + _F(eps))) * size
    bits = random_bits(salt, step, count)
    c0, s0 = held8(m, bits >> np.uint32(16), False)
    c1, s1 = held8(r, bits & np.uint32(0xFFFF), True)
    return p, (c0, c1), (s0, s1)
