"""Cases of the sequence operators and of the decoupled-decay optimizer, each with its plain form.

Three operators of a selective-state-space sequence head and of its training:

* the short causal convolution along time (one filter of 1 to 8 taps a channel, SiLU behind it), for whole sequences, with gradients,
  and for single frames over a kept window;
* the selective scan  h_t = exp(delta_t A) h_{t-1} + delta_t u_t B_t,  y_t = (C_t h_t + D u_t) silu(z_t),  for whole sequences, with
  gradients, and for single frames over a kept state;
* AdamW over all tensors of a model in few launches, its two moments held in 32 bits or in 8 (e4m3 values with one scale a block of
  256, the second as its square root, both rounded stochastically from a counter).

`run` computes them with elementary torch operations where `own` is false and calls the framework where it is true.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ADAMW = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 1e-2, "seed": 1234}
BLOCK = 256             # values that share one scale of an 8-bit state
E4M3_MAX = 448.0
TINY = 2.0 ** -126      # a block whose scale would be below the normal numbers is held as zeros


# ------------------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a bank of 48 live streams, one new frame each: the launch is what it costs
        dict(name="conv step 48 streams", kind="conv_step", n=48, d=1536, k=4, dtype="bf16"),
        # the head of the tagger's third block (53 frames of a 10-second clip, batch 128), a training step
        dict(name="conv train head", kind="conv_train", n=128, t=53, d=256, k=4, dtype="fp32", ragged=False, initial=False, split=True),
        # long recordings of unequal length, continued from a window
        dict(name="conv train long", kind="conv_train", n=4, t=8191, d=2048, k=4, dtype="bf16", ragged=True, initial=True, split=True),
        # one live stream, one frame
        dict(name="scan step one stream", kind="scan_step", n=1, d=256, s=16, g=1, dtype="fp32"),
        # many streams with a wide state: the state's traffic
        dict(name="scan step 256 streams", kind="scan_step", n=256, d=2048, s=64, g=4, dtype="fp16"),
        # one 10-second clip at the front-end's frame rate (431 frames), inference
        dict(name="scan prompt clip", kind="scan_prompt", n=1, t=431, d=512, s=16, g=1, dtype="fp32", ragged=False, initial=False, split=True),
        # long recordings, inference, the state kept for what follows
        dict(name="scan prompt long", kind="scan_prompt", n=2, t=16384, d=2048, s=16, g=1, dtype="bf16", ragged=True, initial=True, split=True),
        # the head of the tagger's third block, a training step
        dict(name="scan train head", kind="scan_train", n=128, t=53, d=256, s=16, g=1, dtype="fp32", ragged=False, initial=False, split=True),
        # long training sequences
        dict(name="scan train long", kind="scan_train", n=8, t=2048, d=1024, s=16, g=1, dtype="bf16", ragged=True, initial=False, split=True),
        # the parameters of the benchmark's six-block tagger (some 230 tensors from 2 numbers to 2.3 million), moments in 32 bits
        dict(name="adamw tagger 32", kind="adamw", bits=32, dtype="fp32", layout="tagger", base=100, growth=1.5, blocks=6),
        # the same with moments in 8 bits
        dict(name="adamw tagger 8", kind="adamw", bits=8, dtype="fp32", layout="tagger", base=100, growth=1.5, blocks=6),
        # few large tensors in 16 bits, moments in 8
        dict(name="adamw large 8", kind="adamw", bits=8, dtype="bf16", layout="even", tensors=12, total=200_000_003),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["conv_step", "conv_train", "conv_prompt", "scan_step", "scan_prompt", "scan_train", "scan_train", "adamw", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "adamw":
        bits = rng.choice([32, 8])
        if rng.random() < 0.5:
            return dict(kind=kind, bits=bits, dtype=dtype, layout="tagger", base=_log(rng, 8, 100), growth=rng.uniform(1.2, 1.5), blocks=rng.randint(2, 6))
        return dict(kind=kind, bits=bits, dtype=dtype, layout="even", tensors=_log(rng, 1, 200), total=_log(rng, 1000, 100_000_000))
    n, d = _log(rng, 1, 256), _log(rng, 5, 2048)
    case = dict(kind=kind, n=n, d=d, dtype=dtype)
    if kind.startswith("conv"):
        case["k"] = rng.randint(1, 8)
        room = 60_000_000 // (n * d)
    else:
        case["s"] = rng.choice([4, 8, 16, 16, 16, 24, 32, 64, rng.randint(1, 64)])
        case["g"] = rng.choice([g for g in (1, 1, 2, 4, 3) if d % g == 0])
        room = 200_000_000 // (n * d * case["s"])
    if kind.endswith("step"):
        return case
    case["t"] = max(1, _log(rng, 1, max(1, min(16384, room))))
    return dict(case, ragged=rng.random() < 0.4, initial=rng.random() < 0.4, split=rng.random() < 0.6)


def _tagger_shapes(base, growth, blocks, classes=80, heads_from=2):
    """Parameter shapes of the 2-d tagger: per block an input norm, the entry convolution, a norm, a PReLU and the residual unit
    (three norms, three PReLUs, convolutions of 1, 9 and 1 taps), then the classifier over the depths of the supervised blocks."""
    shapes, cin, total = [], 2, 0
    for k in range(blocks):
        c = int(growth ** k * base)
        total += c if k >= min(heads_from, blocks - 1) else 0
        shapes += [(cin,), (cin,), (c, cin, 3, 3), (c,)] + [(c,)] * 3
        shapes += [(c, c, 1, 1), (c,), (c,), (c,), (c, c, 3, 3), (c,), (c,), (c,), (c, c, 1, 1), (c,), (c,), (c,)] + [(c,)] * 3
        cin = c
    return shapes + [(total,), (total,), (total, total), (total,), (total,), (total,), (total,), (classes, total), (classes,)]


def _shapes(case):
    if case["layout"] == "tagger":
        return _tagger_shapes(case["base"], case["growth"], case["blocks"])
    count = min(case["tensors"], case["total"])
    cuts = [case["total"] * i // count for i in range(count + 1)]
    return [(hi - lo,) for lo, hi in zip(cuts, cuts[1:])]


def _numel(shape):
    return math.prod(shape)


# ------------------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case, gen):
    if not case["ragged"]:
        return None
    n, t = case["n"], case["t"]
    lengths = torch.randint(max(1, t // 2), t + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)
    lengths[0] = t
    return lengths


def _half(case, gen, dtype):
    """(N, T, D): with `split` the second half of a projection twice as wide, as a gated layer hands it over."""
    n, t, d = case["n"], case["t"], case["d"]
    if case["split"]:
        return torch.randn(n, t, 2 * d, generator=gen, device="cuda").to(dtype)[..., d:]
    return torch.randn(n, t, d, generator=gen, device="cuda").to(dtype)


def _prepare_conv(case, gen, dtype):
    n, d, k = case["n"], case["d"], case["k"]
    s = {"weight": torch.randn(d, k, generator=gen, device="cuda") / math.sqrt(k), "bias": 0.1 * torch.randn(d, generator=gen, device="cuda")}
    window = lambda: torch.randn(n, k - 1, d, generator=gen, device="cuda").to(dtype)  # noqa: E731
    if case["kind"] == "conv_step":
        return dict(s, x=torch.randn(n, d, generator=gen, device="cuda").to(dtype), window=window())
    s["x"] = _half(case, gen, dtype)
    s["lengths"] = _lengths(case, gen)
    s["initial"] = window() if case["initial"] else None
    if case["kind"] == "conv_train":
        s["gy"] = torch.randn(n, case["t"], d, generator=gen, device="cuda").to(dtype)
    return s


def _prepare_scan(case, gen, dtype):
    n, d, st, g = case["n"], case["d"], case["s"], case["g"]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    # time constants between a frame and a thousand, as such heads are initialised, and a little training behind them
    rate = torch.exp(torch.rand(d, generator=gen, device="cuda") * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    s = {"a_log": torch.log(torch.arange(1, st + 1, device="cuda").float()).repeat(d, 1) + 0.1 * randn(d, st),
         "d": 1 + 0.1 * randn(d), "dt_bias": rate + torch.log(-torch.expm1(-rate))}
    if case["kind"] == "scan_step":
        s.update(u=randn(n, d), dt=0.5 * randn(n, d), b=randn(n, g, st), c=randn(n, g, st), z=randn(n, d))
        s = {key: v.to(dtype) if key in ("u", "dt", "b", "c", "z") else v for key, v in s.items()}
        return dict(s, state=0.1 * randn(n, d, st))
    t = case["t"]
    u = randn(n, t, d)
    s["u"] = (u * torch.sigmoid(u)).to(dtype)
    s["dt"] = (0.5 * randn(n, t, d)).to(dtype)
    if case["split"]:        # B and C as the model takes them out of one projection
        bc = randn(n, t, 2 * g * st).to(dtype)
        s["b"], s["c"] = bc[..., :g * st].unflatten(-1, (g, st)), bc[..., g * st:].unflatten(-1, (g, st))
    else:
        s["b"], s["c"] = randn(n, t, g, st).to(dtype), randn(n, t, g, st).to(dtype)
    s["z"] = _half(case, gen, dtype)
    s["lengths"] = _lengths(case, gen)
    s["initial"] = 0.1 * randn(n, d, st) if case["initial"] else None
    if case["kind"] == "scan_train":
        s["gy"] = randn(n, t, d).to(dtype)
    return s


def _prepare_adamw(case, gen, dtype):
    shapes = _shapes(case)
    at, blocks, spans = 0, 0, []
    for shape in shapes:                                    # tensors lie in their buffer as an allocator places them
        count = _numel(shape)
        spans.append((at, count, blocks, -(-count // BLOCK)))
        at += -(-count // 128) * 128
        blocks += -(-count // BLOCK)
    p = torch.zeros(at, device="cuda", dtype=dtype)
    grad, m, v = (torch.zeros(at, device="cuda") for _ in range(3))
    if case["bits"] == 8:
        scales = torch.zeros(2, blocks, device="cuda")
        codes = torch.zeros(2, at, device="cuda", dtype=torch.float8_e4m3fn)
    for shape, (lo, count, block, nb) in zip(shapes, spans):
        part = slice(lo, lo + count)
        p[part] = (0.05 * torch.randn(count, generator=gen, device="cuda")).to(dtype)
        size = torch.exp(2 * torch.randn(count, generator=gen, device="cuda")) * 1e-3       # gradients of one tensor span some decades
        grad[part] = size * torch.randn(count, generator=gen, device="cuda")
        m[part] = 0.3 * size * torch.randn(count, generator=gen, device="cuda")
        v[part] = size.square() * (0.5 + torch.rand(count, generator=gen, device="cuda"))
        if case["bits"] == 8:
            for i, x in enumerate((m[part], v[part].sqrt())):
                rows = torch.nn.functional.pad(x, (0, nb * BLOCK - count)).view(nb, BLOCK)
                scales[i, block:block + nb] = rows.abs().amax(1) / E4M3_MAX
                codes[i, part] = (rows / scales[i, block:block + nb, None]).view(-1)[:count].clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    s = {"step": 100, "p": p, "grad": grad.to(dtype), "params": [], "shapes": shapes, "spans": spans}
    if case["bits"] == 8:
        s.update(codes=codes, scales=scales)
    else:
        s.update(m=m, v=v)
    for shape, (lo, count, _, _) in zip(shapes, spans):
        param = torch.nn.Parameter(p[lo:lo + count].view(shape))
        param.grad = s["grad"][lo:lo + count].view(shape)
        s["params"].append(param)
    if own:
        from freesound_classification_amd.ops.training import FusedAdamW
        s["optimizer"] = FusedAdamW(s["params"], lr=ADAMW["lr"], betas=(ADAMW["beta1"], ADAMW["beta2"]), eps=ADAMW["eps"],
                                    weight_decay=ADAMW["weight_decay"], state_bits=case["bits"], seed=ADAMW["seed"])
        for param, shape, (lo, count, block, nb) in zip(s["params"], shapes, spans):
            if case["bits"] == 8:
                kept = {"exp_avg": codes[0, lo:lo + count].view(shape), "exp_avg_scale": scales[0, block:block + nb],
                        "exp_avg_sq_root": codes[1, lo:lo + count].view(shape), "exp_avg_sq_root_scale": scales[1, block:block + nb]}
            else:
                kept = {"exp_avg": m[lo:lo + count].view(shape), "exp_avg_sq": v[lo:lo + count].view(shape)}
            s["optimizer"].state[param] = dict(kept, step=s["step"])
    return s


def prepare(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    make = _prepare_adamw if case["kind"] == "adamw" else _prepare_conv if case["kind"].startswith("conv") else _prepare_scan
    return dict(make(case, gen, dtype), case=case)


# -------------------------------------------------------------------------------------------------------------------- plain forms
def _mask(lengths, t):
    """(N, T, 1) truth values of the frames that exist, or None."""
    return None if lengths is None else (torch.arange(t, device="cuda") < lengths[:, None])[..., None]


def _kept(x, mask):
    """x in 32 bits, with zeros at the frames that do not exist."""
    x = x.float()
    return x if mask is None else torch.where(mask, x, torch.zeros((), device=x.device))


def _silu_grad(x):
    sig = torch.sigmoid(x)
    return sig * (1 + x * (1 - sig))


def _conv_plain(s):
    x, w, bias, lengths = s["x"], s["weight"], s["bias"], s["lengths"]
    (n, t, d), k = x.shape, w.shape[1]
    mask = _mask(lengths, t)
    before = x.new_zeros(n, k - 1, d).float() if s["initial"] is None else s["initial"].float()
    xin = torch.cat([before, _kept(x, mask)], 1)                                # (N, K - 1 + T, D)
    taps = xin.unfold(1, k, 1)                                                  # (N, T, D, K)
    pre = (taps * w).sum(-1) + bias
    y = _kept(pre * torch.sigmoid(pre), mask).to(x.dtype)
    ends = torch.full((n,), t, device="cuda") if lengths is None else lengths.long()
    where = (ends[:, None] + torch.arange(k - 1, device="cuda"))[..., None].expand(n, k - 1, d)
    if "gy" not in s:
        return {"y": y, "final": xin.gather(1, where).to(x.dtype)}
    dpre = _kept(s["gy"].float() * _silu_grad(pre), mask)
    wide = torch.nn.functional.pad(dpre, (0, 0, k - 1, k - 1))
    dxin = (wide.unfold(1, k, 1) * w.flip(1)).sum(-1)
    out = {"y": y, "dx": dxin[:, k - 1:].to(x.dtype), "dweight": (dpre[..., None] * taps).sum((0, 1)), "dbias": dpre.sum((0, 1))}
    if s["initial"] is not None:
        out["dinitial"] = dxin[:, :k - 1].to(x.dtype)
    if mask is not None:
        out["dx"] = torch.where(mask, out["dx"], torch.zeros((), device="cuda", dtype=x.dtype))
    return out


def _conv_step_plain(s):
    x, window = s["x"], s["window"]
    taps = torch.cat([window, x[:, None]], 1)
    pre = (taps.float().transpose(1, 2) * s["weight"]).sum(-1) + s["bias"]
    window.copy_(taps[:, 1:])
    return {"y": (pre * torch.sigmoid(pre)).to(x.dtype), "window": window}


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))


def _per_channel(x, d):
    """(..., G, S) -> (..., D, S): the D / G channels of a group share its row."""
    return x.float().repeat_interleave(d // x.shape[-2], dim=-2)


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h_{-1} = 0: the pairs (a, b) of twice the span at every turn."""
    span, t = 1, a.shape[1]
    while span < t:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        span *= 2
        if span < t:
            half = span // 2
            a = torch.cat([a[:, :half], a[:, half:] * a[:, :-half]], 1)
    return b


def _scan_plain(s):
    u_in, lengths = s["u"], s["lengths"]
    n, t, d = u_in.shape
    g, st = s["b"].shape[-2:]
    mask = _mask(lengths, t)
    u, z, raw = _kept(u_in, mask), _kept(s["z"], mask), _kept(s["dt"], mask) + s["dt_bias"]
    delta = _kept(_softplus(raw), mask)                                         # 0 where there is no frame: the state stays
    b, c = (_per_channel(_kept(s[key], None if mask is None else mask[..., None]), d) for key in ("b", "c"))
    minus = -torch.exp(s["a_log"])                                              # A
    a = torch.exp(delta[..., None] * minus)                                     # (N, T, D, S)
    drive = (delta * u)[..., None] * b
    if s["initial"] is not None:
        drive[:, 0] += a[:, 0] * s["initial"]
    h = _doubling(a, drive)
    del drive
    inner = (h * c).sum(-1) + s["d"] * u
    y = _kept(inner * z * torch.sigmoid(z), mask).to(u_in.dtype)
    if "gy" not in s:
        return {"y": y, "final": h[:, -1].contiguous()}
    gy = _kept(s["gy"], mask)
    dinner = gy * z * torch.sigmoid(z)
    out = {"y": y, "dz": (gy * inner * _silu_grad(z)).to(u_in.dtype)}
    shared = lambda x: x.unflatten(2, (g, d // g)).sum(3).to(u_in.dtype)  # noqa: E731
    out["dc"] = shared(h * dinner[..., None])
    before = torch.zeros_like(h[:, :1]) if s["initial"] is None else s["initial"][:, None]
    ah = a * torch.cat([before, h[:, :-1]], 1)                                  # exp(delta A) h_{t-1}
    del h
    nexts = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    gh = _doubling(nexts.flip(1), (c * dinner[..., None]).flip(1)).flip(1)      # dL/dh_t
    del nexts
    out["db"] = shared(gh * (delta * u)[..., None])
    if s["initial"] is not None:
        out["dinitial"] = a[:, 0] * gh[:, 0]
    del a
    gb = (gh * b).sum(-1)
    gah = gh * ah
    del gh, ah
    out["da_log"] = (gah * delta[..., None]).sum((0, 1)) * minus
    draw_ = ((gah * minus).sum(-1) + u * gb) * torch.sigmoid(raw)
    out["ddt"] = _kept(draw_, mask).to(u_in.dtype)
    out["du"] = (delta * gb + s["d"] * dinner).to(u_in.dtype)
    out["dd"] = (dinner * u).sum((0, 1))
    out["ddt_bias"] = _kept(draw_, mask).sum((0, 1))
    return out


def _scan_step_plain(s):
    d = s["u"].shape[-1]
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    a = torch.exp(delta[..., None] * -torch.exp(s["a_log"]))
    s["state"].copy_(a * s["state"] + (delta * s["u"].float())[..., None] * _per_channel(s["b"], d))
    z = s["z"].float()
    inner = (s["state"] * _per_channel(s["c"], d)).sum(-1) + s["d"] * s["u"].float()
    return {"y": (inner * z * torch.sigmoid(z)).to(s["u"].dtype), "state": s["state"]}


def _mix(x):
    """A bijection of 32-bit numbers whose bits all depend on all bits."""
    x = ((x ^ (x >> 16)) * 0x9E3779B9) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xB7E15163) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(ordinal, step, count):
    """32 bits for each element of the optimizer's tensor `ordinal` at this step: the upper 16 round the first moment, the lower the second."""
    key = _mix((_mix((ADAMW["seed"] + ordinal) & 0xFFFFFFFF) + step) & 0xFFFFFFFF)
    return _mix(torch.arange(count, device="cuda") ^ key)


def _held(x, bits16):
    """(e4m3 values, scales of the blocks of 256) for x: rounded down or up with the probability of the remainder, a value other than 0 of a
    block that is not all 0 never to 0 where it has no sign to lose (x >= 0 throughout); not-finite values stay out of the block's maximum."""
    count = x.numel()
    rows = torch.nn.functional.pad(x.view(-1), (0, -count % BLOCK)).view(-1, BLOCK)
    top = torch.where(torch.isfinite(rows), rows.abs(), torch.zeros((), device="cuda")).amax(1)
    scale = top / E4M3_MAX
    dead = scale < TINY
    scale = torch.where(dead, torch.zeros((), device="cuda"), scale)
    inverse = torch.where(dead, torch.zeros((), device="cuda"), E4M3_MAX / torch.where(dead, torch.ones((), device="cuda"), top))
    y = (rows * inverse[:, None]).view(-1)[:count]
    size, pattern = y.abs(), y.abs().view(torch.int32).long()
    normal = ((pattern + (bits16 << 4)) >> 20) - (120 << 3)
    small = torch.floor(size * 512 + bits16.float() * 2.0 ** -16).long()
    code = torch.clamp(torch.where(size >= 2.0 ** -6, normal, small), max=0x7E)
    return code, y, scale


def _e4m3(code, y):
    code = torch.where(torch.isfinite(y), code | torch.where(torch.signbit(y), 0x80, 0), 0x7F)
    return code.to(torch.uint8).view(torch.float8_e4m3fn)


def _adamw_plain(s):
    s["step"] += 1
    step, bits = s["step"], s["case"]["bits"]
    b1, b2 = ADAMW["beta1"], ADAMW["beta2"]
    size, root = ADAMW["lr"] / (1 - b1 ** step), 1 / math.sqrt(1 - b2 ** step)
    for i, (lo, count, block, nb) in enumerate(s["spans"]):
        part, blocks = slice(lo, lo + count), slice(block, block + nb)
        p, g = s["p"][part].float(), s["grad"][part].float()
        if bits == 32:
            m, v = s["m"][part], s["v"][part]
        else:
            m, v = (s["codes"][j, part].float() * s["scales"][j, blocks].repeat_interleave(BLOCK)[:count] for j in (0, 1))
            v = v * v
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * g) * (1 - b2)
        r = v.sqrt()
        p = p * (1 - ADAMW["lr"] * ADAMW["weight_decay"]) - (m / (r * root + ADAMW["eps"])) * size
        s["p"][part] = p.to(s["p"].dtype)
        if bits == 32:
            s["m"][part], s["v"][part] = m, v
            continue
        random = _random_bits(i, step, count)
        code, y, s["scales"][0, blocks] = _held(m, random >> 16)
        s["codes"][0, part] = _e4m3(code, y)
        code, y, s["scales"][1, blocks] = _held(r, random & 0xFFFF)
        s["codes"][1, part] = _e4m3(torch.where((code == 0) & (y > 0), 1, code), y)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    if s["case"]["bits"] == 32:
        return {"p": s["p"], "m": s["m"], "v": s["v"]}
    return {"p": s["p"], "codes": s["codes"], "scales": s["scales"]}


# ---------------------------------------------------------------------------------------------------------------- the framework's
def _conv_own(s):
    from freesound_classification_amd import functional as F
    if "gy" not in s:
        y, final = F.causal_conv(s["x"], s["weight"], s["bias"], activation="silu", lengths=s["lengths"], initial=s["initial"], return_final=True)
        return {"y": y, "final": final}
    names = ["x", "weight", "bias"] + (["initial"] if s["initial"] is not None else [])
    leaves = {key: s[key].detach().requires_grad_() for key in names}
    y = F.causal_conv(leaves["x"], leaves["weight"], leaves["bias"], activation="silu", lengths=s["lengths"], initial=leaves.get("initial"))
    grads = torch.autograd.grad(y, list(leaves.values()), s["gy"])
    return dict({"d" + key: g for key, g in zip(names, grads)}, y=y)


def _scan_own(s):
    from freesound_classification_amd import functional as F
    if "gy" not in s:
        y, final = F.selective_scan(s["u"], s["dt"], s["a_log"], s["b"], s["c"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"], softplus=True,
                                    lengths=s["lengths"], initial=s["initial"], return_final=True)
        return {"y": y, "final": final}
    names = ["u", "dt", "a_log", "b", "c", "d", "z", "dt_bias"] + (["initial"] if s["initial"] is not None else [])
    leaves = {key: s[key].detach().requires_grad_() for key in names}
    y = F.selective_scan(leaves["u"], leaves["dt"], leaves["a_log"], leaves["b"], leaves["c"], d=leaves["d"], z=leaves["z"],
                         dt_bias=leaves["dt_bias"], softplus=True, lengths=s["lengths"], initial=leaves.get("initial"))
    grads = torch.autograd.grad(y, list(leaves.values()), s["gy"])
    return dict({"d" + key: g for key, g in zip(names, grads)}, y=y)


def _step_own(s):
    from freesound_classification_amd import functional as F
    if s["case"]["kind"] == "conv_step":
        return {"y": F.causal_conv_step(s["x"], s["window"], s["weight"], s["bias"], activation="silu"), "window": s["window"]}
    y = F.selective_scan_step(s["u"], s["dt"], s["a_log"], s["b"], s["c"], s["state"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"], softplus=True)
    return {"y": y, "state": s["state"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        if kind == "adamw":
            state["optimizer"].step()
            return _adamw_outputs(state)
        return _step_own(state) if kind.endswith("step") else _conv_own(state) if kind.startswith("conv") else _scan_own(state)
    if kind == "adamw":
        return _adamw_plain(state)
    if kind.endswith("step"):
        return _conv_step_plain(state) if kind == "conv_step" else _scan_step_plain(state)
    return _conv_plain(state) if kind.startswith("conv") else _scan_plain(state)


def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "fp32" else 2
    if kind == "adamw":
        count = sum(_numel(shape) for shape in _shapes(case))
        held = 2 * (1 + 4 / BLOCK) if case["bits"] == 8 else 8
        return {"bytes": count * (3 * size + 2 * held), "flops": 16 * count}
    n, d, t = case["n"], case["d"], case.get("t", 1)
    frames = n * t * d
    if kind.startswith("conv"):
        k = case["k"]
        passes, flops = (4, 6 * k + 16) if kind == "conv_train" else (2, 2 * k + 4)
        window = n * (k - 1) * d * size * (2 if kind != "conv_train" else 2 * case["initial"])
        return {"bytes": passes * frames * size + window + 8 * d * (k + 1), "flops": flops * frames}
    st, g = case["s"], case["g"]
    rows, states = n * t * g * st, n * d * st
    if kind == "scan_train":
        return {"bytes": (8 * frames + 4 * rows) * size + 8 * d * (st + 2) + 8 * states * case["initial"], "flops": frames * (29 * st + 40)}
    kept = 8 * states if kind == "scan_step" or case["initial"] else 4 * states
    return {"bytes": (4 * frames + 2 * rows) * size + kept + 4 * d * (st + 2), "flops": frames * (7 * st + 16)}


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_conv(case, s):
    k, t = case["k"], case.get("t", 1)
    if case["kind"] == "conv_step":
        rows = torch.cat([s["window"], s["x"][:, None]], 1).double()
        pre = s["bias"].double() + sum(rows[:, i] * s["weight"][:, i].double() for i in range(k))
        return {"y": torch.nn.functional.silu(pre), "window": rows[:, 1:]}
    names = ["x", "weight", "bias"] + (["initial"] if s["initial"] is not None else [])
    leaves = {key: s[key].double().requires_grad_("gy" in s) for key in names}
    there = torch.ones(case["n"], t, 1, device="cuda", dtype=torch.bool) if s["lengths"] is None else _mask(s["lengths"], t)
    before = leaves["initial"] if "initial" in leaves else torch.zeros(case["n"], k - 1, case["d"], device="cuda", dtype=torch.float64)
    rows = torch.cat([before, leaves["x"]], 1)
    pre = leaves["bias"] + sum(rows[:, i:i + t] * leaves["weight"][:, i] for i in range(k))
    y = torch.nn.functional.silu(pre) * there
    if "gy" not in s:
        ends = [t] * case["n"] if s["lengths"] is None else s["lengths"].tolist()
        return {"y": y, "final": torch.stack([rows[i, end:end + k - 1] for i, end in enumerate(ends)])}
    grads = torch.autograd.grad(y, list(leaves.values()), s["gy"].double())
    return dict({"d" + key: g for key, g in zip(names, grads)}, y=y.detach())


def _exact_scan(case, s):
    step, groups = case["kind"] == "scan_step", case["g"]
    if step:                                   # a sequence of one frame that begins at the kept state
        s = dict({key: s[key][:, None] if key in ("u", "dt", "b", "c", "z") else s[key] for key in s}, initial=s["state"], lengths=None)
    names = ["u", "dt", "a_log", "b", "c", "d", "z", "dt_bias"] + (["initial"] if s["initial"] is not None else [])
    train = "gy" in s
    leaves = {key: s[key].double().requires_grad_(train) for key in names}
    n, t, d = s["u"].shape
    delta = torch.nn.functional.softplus(leaves["dt"] + leaves["dt_bias"], threshold=40)
    rate = -leaves["a_log"].exp()
    h = leaves.get("initial", torch.zeros(n, d, case["s"], device="cuda", dtype=torch.float64)).unflatten(1, (groups, d // groups))
    rate = rate.unflatten(0, (groups, d // groups))
    ends = None if s["lengths"] is None else s["lengths"].long()
    inner = []
    frames = zip(delta.unbind(1), (delta * leaves["u"]).unbind(1), leaves["b"].unbind(1), leaves["c"].unbind(1))
    for i, (dl, du, b, c) in enumerate(frames):
        dl, du = dl.unflatten(1, (groups, d // groups)), du.unflatten(1, (groups, d // groups))
        new = torch.exp(dl[..., None] * rate) * h + du[..., None] * b[:, :, None]
        h = new if ends is None else torch.where((ends > i)[:, None, None, None], new, h)
        inner.append((h * c[:, :, None]).sum(-1).flatten(1))
    y = (torch.stack(inner, 1) + leaves["d"] * leaves["u"]) * torch.nn.functional.silu(leaves["z"])
    if ends is not None:
        y = y * _mask(ends, t)
    if not train:
        h = h.flatten(1, 2)
        return {"y": y[:, 0], "state": h} if step else {"y": y, "final": h}
    grads = torch.autograd.grad(y, list(leaves.values()), s["gy"].double())
    return dict({"d" + key: g for key, g in zip(names, grads)}, y=y.detach())


def _exact_adamw(case, s):
    step = s["step"] + 1
    b1, b2, lr = ADAMW["beta1"], ADAMW["beta2"], ADAMW["lr"]
    bits = case["bits"]
    new = {key: torch.zeros_like(s["p"], dtype=torch.float64) for key in ("p", "m", "v")}
    scales = torch.zeros_like(s["scales"], dtype=torch.float64) if bits == 8 else None
    for i, (lo, count, block, nb) in enumerate(s["spans"]):
        part = slice(lo, lo + count)
        p, g = s["p"][part].double(), s["grad"][part].double()
        if bits == 8:
            each = torch.arange(count, device="cuda") // BLOCK + block
            m, v = s["codes"][0, part].double() * s["scales"][0, each], (s["codes"][1, part].double() * s["scales"][1, each]) ** 2
        else:
            m, v = s["m"][part].double(), s["v"][part].double()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        update = lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + ADAMW["eps"])
        new["p"][part] = p - lr * ADAMW["weight_decay"] * p - update
        if bits == 32:
            new["m"][part], new["v"][part] = m, v
            continue
        random = _random_bits(i, step, count)
        for j, (key, x, bits16) in enumerate((("m", m, random >> 16), ("v", v.sqrt(), random & 0xFFFF))):
            top = torch.zeros(blocks_of(count), device="cuda", dtype=torch.float64).scatter_reduce(0, each - block, x.abs(), "amax")
            scales[j, block:block + nb] = top / E4M3_MAX
            y = x * (E4M3_MAX / top)[each - block]
            grid = 2.0 ** (torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4).double()        # the distance of e4m3 values around y
            held = (torch.floor(y.abs() / grid + bits16 * 2.0 ** -16) * grid).clamp(max=E4M3_MAX)
            held = held.clamp(min=2.0 ** -9) if j else held
            new[key][part] = held * torch.sign(y)
    if bits == 32:
        return new
    return {"p": new["p"], "codes": torch.stack([new["m"], new["v"]]), "scales": scales}


def blocks_of(count):
    return -(-count // BLOCK)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adamw":
        return _exact_adamw(case, s)
    return _exact_conv(case, s) if case["kind"].startswith("conv") else _exact_scan(case, s)
