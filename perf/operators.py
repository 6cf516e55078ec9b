"""Timed cases of the layer norm (forward, backward) and of the AdamW step with 8-bit moments.

`run` computes an operator in elementary torch operations (fp32, sums over rows in fp64) or, with `own` set, calls the
framework's kernels on the same data.  The 8-bit moments: 64 elements share a biased exponent e; a first moment is
sign | 4 exponent bits | 3 mantissa bits, a second moment 5 exponent bits | 3 mantissa bits, both relative to e, with
subnormals; a value is rounded stochastically with 20 bits of a hash of (seed, step, index in its tensor).  They are
returned as the values they stand for, in bfloat16, which holds each of them exactly.
"""
import math
import random

import torch

own = False

EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 1e-4
BLOCK = 64


# ----------------------------------------------------------------------------- the cases

def listed():
    return [
        # deepest level of a two-level RepUNet on a 32x32 image: one call of a latency-bound evaluation
        {"name": "ln_fwd_small", "op": "ln_fwd", "rows": 64, "channels": 32, "branches": 3, "relu": True, "dtype": "bf16", "slice": False},
        # first level of the two-kernel-size RepUNet, batch 8 of 512x512 slices, written into the skip half of the concat buffer
        {"name": "ln_fwd_repunet", "op": "ln_fwd", "rows": 8 * 512 * 512, "channels": 64, "branches": 6, "relu": True, "dtype": "bf16", "slice": True},
        # token rows of a wide layer, plain layer norm
        {"name": "ln_fwd_wide", "op": "ln_fwd", "rows": 8192, "channels": 4096, "branches": 1, "relu": False, "dtype": "bf16", "slice": False},
        # fp32 training (amp off) with an odd width: no row is aligned
        {"name": "ln_fwd_odd_f32", "op": "ln_fwd", "rows": 50001, "channels": 333, "branches": 1, "relu": False, "dtype": "f32", "slice": False},
        # backward of a small fp32 block, ragged row count
        {"name": "ln_bwd_small", "op": "ln_bwd", "rows": 196, "channels": 120, "branches": 3, "relu": True, "dtype": "f32", "slice": False},
        # backward of the first level, the largest call of a RepUNet step
        {"name": "ln_bwd_repunet", "op": "ln_bwd", "rows": 8 * 512 * 512, "channels": 64, "branches": 6, "relu": True, "dtype": "bf16", "slice": False},
        # bottleneck of the same network: 1024 channels on 32x32
        {"name": "ln_bwd_deep", "op": "ln_bwd", "rows": 8 * 32 * 32, "channels": 1024, "branches": 6, "relu": True, "dtype": "bf16", "slice": False},
        # token rows of a wide layer, ragged count
        {"name": "ln_bwd_wide", "op": "ln_bwd", "rows": 4099, "channels": 5120, "branches": 1, "relu": False, "dtype": "bf16", "slice": False},
        # optimizer step of a two-level U-Net (features 16, 32): launch-bound
        {"name": "adamw8_small", "op": "adamw8", "model": "unet", "features": "16,32", "clip": 0.5, "shift": 0},
        # the benchmark's U-Net, 31 M parameters, gradients clipped
        {"name": "adamw8_unet", "op": "adamw8", "model": "unet", "features": "64,128,256,512", "clip": 0.37, "shift": 0},
        # RepUNet with kernel sizes 3 and 5: 160 M parameters in 334 tensors, not clipped
        {"name": "adamw8_repunet", "op": "adamw8", "model": "repunet", "features": "64,128,256,512", "clip": 1.0, "shift": 0},
        # many ragged tensors; parameters and gradients are views that start on any 4-byte boundary
        {"name": "adamw8_ragged", "op": "adamw8", "model": "list", "tensors": 300, "elements": 5000011, "sizes": 1, "clip": 0.8, "shift": 3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "adamw8"])
    if op == "adamw8":
        model = rng.choice(["unet", "repunet", "list"])
        case = {"op": op, "model": model, "clip": rng.choice([1.0, round(rng.uniform(0.05, 0.95), 3)]), "shift": rng.randrange(4)}
        if model == "list":
            tensors = _log(rng, 1, 400)
            return {**case, "tensors": tensors, "elements": _log(rng, 2 * tensors, 1.2e8), "sizes": rng.randrange(1 << 20)}
        width = 8 * rng.randint(1, 8 if model == "unet" else 4)
        return {**case, "features": ",".join(str(width << i) for i in range(rng.randint(1, 4)))}
    branches = rng.choice([1, 1, 2, 3, 6, 8])
    channels = _log(rng, 8, 8192)
    rows = _log(rng, 1, min(1 << 21, (1 << 28) // (channels * (branches + 1))))
    return {"op": op, "rows": rows, "channels": channels, "branches": branches, "relu": rng.random() < 0.5,
            "dtype": rng.choice(["bf16", "f32"]), "slice": rng.random() < 0.3}


# ----------------------------------------------------------------------------- shapes

def _unet_shapes(features, kernel_sizes=None):
    """Parameter shapes of the U-Net (or, with kernel sizes, of the multi-branch RepUNet) in registration order."""
    def conv(i, o):
        if kernel_sizes is None:
            return [(o, i, 3, 3), (o,), (o,), (o,)]
        return [s for k in kernel_sizes for kk in ((k, 1), (1, k), (k, k)) for s in ((o, i) + kk, (o,), (o,))]

    def block(i, o):
        return conv(i, o) + conv(o, o)
    ins = [1] + features[:-1]
    shapes = [s for f in reversed(features) for s in [(2 * f, f, 2, 2), (f,)] + block(2 * f, f)]
    shapes += [s for i, o in zip(ins, features) for s in block(i, o)]
    return shapes + block(features[-1], 2 * features[-1]) + [(2, features[0], 1, 1), (2,)]


def _numels(case):
    if case["model"] == "list":
        rng = random.Random(case["sizes"])
        w = [math.exp(rng.uniform(0, 6)) for _ in range(case["tensors"])]
        return [max(1, int(case["elements"] * x / sum(w))) for x in w]
    features = [int(f) for f in case["features"].split(",")]
    return [math.prod(s) for s in _unet_shapes(features, [3, 5] if case["model"] == "repunet" else None)]


# ----------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g = _gen(seed)
    return _prepare_adamw8(case, g, seed) if case["op"] == "adamw8" else _prepare_ln(case, g)


def _rand(shape, g, dtype, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _prepare_ln(case, g):
    """Conv outputs of each branch (their scales and means differ), weights near 1; activations are [1, 1, rows, channels]."""
    M, C, nb = case["rows"], case["channels"], case["branches"]
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    s = {"case": case, "zs": [_rand((1, 1, M, C), g, dt, 0.5 + 0.25 * b, 0.3 * b - 0.4) for b in range(nb)],
         "gammas": [_rand(C, g, torch.float32, 0.2, 1.0) for _ in range(nb)],
         "betas": [_rand(C, g, torch.float32, 0.2) for _ in range(nb)]}
    ld, off = (2 * C, C) if case["slice"] else (C, 0)
    if case["op"] == "ln_fwd":
        if case["slice"]:
            s["ybuf"], s["off"] = torch.empty((1, 1, M, ld), dtype=dt, device="cuda"), off
    else:
        s["dybuf"], s["off"] = _rand((1, 1, M, ld), g, dt, 0.01), off
        if case["relu"]:
            s["y"] = _plain_ln_fwd(s)
    return s


def _prepare_adamw8(case, g, seed):
    """A training state some steps in: every tensor starts on a block of 64 of the flat buffers (parameters and gradients
    `shift` floats later), as FusedAdamW lays its moments out."""
    n = _numels(case)
    blocks = [-(-k // BLOCK) for k in n]
    total, starts = sum(blocks), [0]
    for b in blocks:
        starts.append(starts[-1] + b)
    shift, pad = case["shift"], total * BLOCK
    tensor = torch.repeat_interleave(torch.arange(len(n), device="cuda"), torch.tensor(blocks, device="cuda"))
    first = torch.tensor(starts[:-1], device="cuda")[tensor]
    block = torch.arange(total, device="cuda") - first                        # index of each block in its tensor
    live = block.view(-1, 1) * BLOCK + torch.arange(BLOCK, device="cuda") < torch.tensor(n, device="cuda")[tensor].view(-1, 1)
    size = torch.exp(torch.randn((len(n), 1), generator=g, device="cuda"))[tensor] * 1e-3        # gradients of each tensor
    per = torch.exp(torch.randn((total, BLOCK), generator=g, device="cuda")) * size * live       # and of each weight
    m0 = torch.randn((total, BLOCK), generator=g, device="cuda") * per * 0.3
    v0 = per * per * (0.5 + torch.rand((total, BLOCK), generator=g, device="cuda"))
    half = torch.full((1,), 1 << 19, dtype=torch.int64, device="cuda")
    (m, em), (v, ev) = _encode(m0, 15, half), _encode(v0, 31, half)
    p = torch.zeros(pad + 4, device="cuda")
    p[shift:shift + pad] = (torch.randn((total, BLOCK), generator=g, device="cuda") * 0.05 * live).view(-1)
    grad = torch.zeros(pad + 4, device="cuda")
    grad[shift:shift + pad] = (torch.randn((total, BLOCK), generator=g, device="cuda") * per).view(-1)
    del per, m0, v0, live
    spans = list(zip(starts[:-1], n))
    return {"case": case, "seed": seed & 0x7fffffff, "step": 100, "block": block, "p": p[shift:shift + pad], "grad": grad[shift:shift + pad],
            "m": m.view(-1), "v": v.view(-1), "em": em.view(-1), "ev": ev.view(-1),
            "norm": torch.tensor([1.0, case["clip"]], device="cuda"),
            "ps": [p[shift + s * BLOCK:shift + s * BLOCK + k] for s, k in spans],
            "gs": [grad[shift + s * BLOCK:shift + s * BLOCK + k] for s, k in spans]}


# ----------------------------------------------------------------------------- layer norm, plain

def _xhat(z):
    """((z - mean) / std, 1 / std) over the last axis."""
    z = z.float()
    d = z - z.sum(-1, keepdim=True) / z.shape[-1]
    rstd = 1.0 / torch.sqrt((d * d).sum(-1, keepdim=True) / z.shape[-1] + EPS)
    return d * rstd, rstd


def _plain_ln_fwd(s):
    y = sum(_xhat(z)[0] * g + b for z, g, b in zip(s["zs"], s["gammas"], s["betas"]))
    y = torch.where(y < 0, 0.0, y) if s["case"]["relu"] else y
    return y.to(s["zs"][0].dtype)


def _plain_ln_bwd(s):
    C = s["case"]["channels"]
    u = s["dybuf"][..., s["off"]:s["off"] + C].float()
    u = torch.where(s["y"].float() <= 0, 0.0, u) if s["case"]["relu"] else u

    def branch(z, gamma):
        x, rstd = _xhat(z)
        w = u * gamma
        dz = rstd * (w - w.sum(-1, keepdim=True) / C - x * ((w * x).sum(-1, keepdim=True) / C))
        return dz.to(z.dtype), (u * x).view(-1, C).sum(0, dtype=torch.float64).float()
    out = [branch(z, gamma) for z, gamma in zip(s["zs"], s["gammas"])]
    db = u.reshape(-1, C).sum(0, dtype=torch.float64).float()
    return {"dz": [o[0] for o in out], "dgamma": [o[1] for o in out], "dbeta": [db] * len(out)}


# ----------------------------------------------------------------------------- AdamW with 8-bit moments, plain

def _dither(block, seed, step):
    """([blocks, 64], [blocks, 64]) 20-bit numbers for the first and the second moment."""
    key = (seed * 0x9E3779B97F4A7C15 + step * 0x6A09E667F3BCC909) & (2 ** 64 - 1)
    key = (((key ^ (key >> 31)) * 0x9E3779B97F4A7C15) & (2 ** 64 - 1)) >> 32
    i = block.view(-1, 1) * BLOCK + torch.arange(BLOCK, device=block.device)
    h = ((i & 0xffffffff) * 0x9E3779B9 + (i >> 32) * 0xBB67AE85 + key) & 0xffffffff
    h = ((h ^ (h >> 15)) * 0x6A09E667) & 0xffffffff
    h = h ^ (h >> 16)
    return ((h & 0xffff) << 4) | 8, ((h >> 16) << 4) | 8


def _bits(x):
    return x.abs().view(torch.int32).long()


def _power(e):
    """2^e in fp64."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x, top, dither):
    """[blocks, 64] fp32 -> (codes, exponents [blocks, 1]), uint8; top = 15: signed first moment, 31: second moment."""
    e = ((_bits(x).amax(-1, keepdim=True) + 0xfffff) >> 23).clamp(32, 255)
    scaled = torch.where(e < 255, (x.abs().double() * _power(top - e)).float(), 0.0)
    c = torch.where(e < 255, (_bits(scaled) + dither) >> 20, 0)
    if top == 31:
        c = torch.where((x > 0) & (e < 255) & (c == 0), 1, c)
    else:
        c = torch.where((x < 0) & (e < 255), c | 128, c)
    return c.to(torch.uint8), e.to(torch.uint8)


def _decode(c, e, top):
    c, e = c.view(-1, BLOCK).int(), e.view(-1, 1).int()
    mag = ((c if top == 31 else c & 127) << 20).view(torch.float32)
    x = (mag.double() * _power(e - top)).float()
    x = x if top == 31 else torch.where(c >= 128, -x, x)
    return torch.where(e == 255, float("nan"), x)


def _plain_adamw8(s):
    step = s["step"]
    omb1, b2, omb2 = 1 - BETA1, BETA2, 1 - BETA2
    shape = s["m"].view(-1, BLOCK).shape
    g = s["grad"].view(shape) * s["norm"][1]
    p = s["p"].view(shape)
    m, v = _decode(s["m"], s["em"], 15), _decode(s["v"], s["ev"], 31)
    m = m + (g - m) * omb1
    v = v * b2 + (omb2 * g) * g
    size = LR / (1 - BETA1 ** step)
    p.copy_(p * (1 - LR * DECAY) - size * (m / (torch.sqrt(v) / math.sqrt(1 - BETA2 ** step) + ADAM_EPS)))
    dm, dv = _dither(s["block"], s["seed"], step)
    for x, top, d, code, exponent in ((m, 15, dm, s["m"], s["em"]), (v, 31, dv, s["v"], s["ev"])):
        c, e = _encode(x, top, d)
        code.copy_(c.view(-1))
        exponent.copy_(e.view(-1))
    return {"p": s["p"], "m": _decode(s["m"], s["em"], 15).bfloat16().view(-1), "v": _decode(s["v"], s["ev"], 31).bfloat16().view(-1)}


# ----------------------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        return {"ln_fwd": _own_ln_fwd, "ln_bwd": _own_ln_bwd, "adamw8": _own_adamw8}[op](s)
    if op == "ln_bwd":
        return _plain_ln_bwd(s)
    if op == "adamw8":
        s["step"] += 1
        return _plain_adamw8(s)
    y = _plain_ln_fwd(s)
    if s["case"]["slice"]:
        view = s["ybuf"][..., s["off"]:]
        view.copy_(y)
        return view
    return y


def _own_ln_fwd(s):
    from unet_amd import ops
    C, zs = s["case"]["channels"], s["zs"]
    if s["case"]["slice"]:
        y = ops.Act(s["ybuf"], s["off"], C)
    else:
        y = ops.Act(torch.empty_like(zs[0]), 0, C)
    ops.layer_norm_fwd([ops.Act(z, 0, C) for z in zs], s["gammas"], s["betas"], y, relu=s["case"]["relu"], eps=EPS)
    return y.buf[..., y.off:y.off + C]


def _own_ln_bwd(s):
    from unet_amd import ops
    C = s["case"]["channels"]
    out = ops.layer_norm_bwd(ops.Act(s["dybuf"], s["off"], C), [ops.Act(z, 0, C) for z in s["zs"]], s["gammas"],
                             y=ops.Act(s["y"], 0, C) if s["case"]["relu"] else None, eps=EPS)
    return {"dz": [o[0].buf for o in out], "dgamma": [o[1] for o in out], "dbeta": [o[2] for o in out]}


def _own_adamw8(s):
    from unet_amd import ops
    s["step"] += 1
    ops.adamw8_step(s["ps"], s["gs"], s["m"], s["v"], s["em"], s["ev"], s["norm"], False, LR, BETA1, BETA2, ADAM_EPS, DECAY,
                    s["step"], seed=s["seed"])
    return {"p": s["p"], "m": ops.moment8_decode(s["m"], s["em"], signed=True, dtype=torch.bfloat16),
            "v": ops.moment8_decode(s["v"], s["ev"], signed=False, dtype=torch.bfloat16)}


# ----------------------------------------------------------------------------- work

def work(case):
    if case["op"] == "adamw8":
        n = sum(_numels(case))
        # p and its gradient in, p out, both codes in and out with an exponent per 64, and the two moments as bfloat16
        return {"bytes": n * (12 + 4 + 4 / BLOCK + 4), "flops": n * 20}
    M, C, nb, size = case["rows"], case["channels"], case["branches"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "ln_fwd":
        return {"bytes": M * C * (nb + 1) * size + 8 * nb * C, "flops": M * C * nb * 8}
    return {"bytes": M * C * (2 * nb + 1 + case["relu"]) * size + 12 * nb * C, "flops": M * C * nb * 16}


# ----------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw8":
        return _exact_adamw8(s)
    C = case["channels"]
    stats = [torch.var_mean(z.double(), dim=-1, correction=0, keepdim=True) for z in s["zs"]]
    if case["op"] == "ln_fwd":
        y = 0.0
        for z, (var, mean), g, b in zip(s["zs"], stats, s["gammas"], s["betas"]):
            y = y + (z.double() - mean) * (var + EPS).rsqrt() * g.double() + b.double()
        return y.clamp_min(0) if case["relu"] else y
    u = s["dybuf"][..., s["off"]:s["off"] + C].double()
    if case["relu"]:
        u = u * (s["y"] > 0)
    out = {"dz": [], "dgamma": [], "dbeta": []}
    for z, (var, mean), g in zip(s["zs"], stats, s["gammas"]):
        std = (var + EPS).sqrt()
        x = (z.double() - mean) / std
        dx = u * g.double()
        out["dz"].append((dx - dx.mean(-1, keepdim=True) - x * (dx * x).mean(-1, keepdim=True)) / std)
        out["dgamma"].append((u * x).sum((0, 1, 2)))
        out["dbeta"].append(u.sum((0, 1, 2)))
    return out


def _exact_adamw8(s):
    """The parameters after one step; the moments' 8-bit values have no 64-bit counterpart (they are rounded at random)."""
    c = torch.arange(256, dtype=torch.float64, device="cuda")

    def table(bits):                                                          # code -> value relative to 2^(e-127)
        mag = c % 2 ** bits
        field, frac = torch.div(mag, 8, rounding_mode="floor"), mag % 8
        top = 2 ** (bits - 3) - 1
        val = torch.where(field > 0, (1 + frac / 8) * 2.0 ** (field - top), frac / 8 * 2.0 ** (1 - top))
        return torch.where(c >= 2 ** bits, -val, val)
    unit = [2.0 ** (s[k].double() - 127).repeat_interleave(BLOCK) for k in ("em", "ev")]
    m, v = table(7)[s["m"].long()] * unit[0], table(8)[s["v"].long()] * unit[1]
    g = s["grad"].double() * float(s["norm"][1])
    t = s["step"] + 1
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    mh, vh = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = s["p"].double() * (1 - LR * DECAY) - LR * mh / (vh.sqrt() + ADAM_EPS)
    return {"p": p, "m": None, "v": None}
