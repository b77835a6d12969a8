"""Cases of the optimizer's operators over many tensors: the global gradient norm with clipping, and the AdamW step with its
moments in 32 bits or in 8.

``run`` makes ONE pass.  With ``own`` set it makes the calls a training program makes (``vae_amd.optim``); otherwise it
computes the same operators from elementary torch operations on the arenas that hold the tensors.

Layout.  The tensors of a case lie in one arena; each starts on a multiple of 256 elements, the padding holds zeros and
stays zero.  Moments have the same layout, so element k of a moment belongs to element k of the parameter arena.

8-bit moments.  Blocks of 256 elements of one tensor.  The fp32 bit pattern of a magnitude shifted right by 20 is its level (8 levels
per octave); a code c > 0 stands for level (base + c) of its block, code 0 for zero.  exp_avg: a sign bit and codes up to 127;
exp_avg_sq: codes up to 254, and no positive value is stored as zero.  Rounding adds d in [0, 2^20) to the bits before the shift; d is
the top 20 bits of (index * A + step * B) mod 2^32, which for every element is equidistributed over the steps.

bf16 parameters.  The parameter and a 16-bit remainder together are the magnitude bits of a 32-bit master value.
"""
import math
import random

import torch

own = False

LR, BETA1, BETA2, EPS, WEIGHT_DECAY, MAX_NORM = 1e-4, 0.9, 0.999, 1e-8, 0.01, 1.0      # the optimizer's defaults, the loop's clip
BLOCK = 256
A, B_M, B_V = 0x9E3779B9, 0xBB67AE85, 0x6A09E667      # fractional parts of the golden ratio, sqrt 3, sqrt 2, times 2^32


# ------------------------------------------------------------------------------------------------ cases
def _double_conv(ci, co):
    return [9 * ci * co, co, co, co, 9 * co * co, co, co, co]


def _module_sizes(module):
    """numbers of elements of a module's parameters, in its own order"""
    if module == "block":          # the GroupNorm double conv, 3 -> 64
        return _double_conv(3, 64)
    if module == "conv32":         # VAEConv(3, 3, 128, image 32): the headline model, 52 tensors
        n = _double_conv(3, 64) + _double_conv(64, 128) + _double_conv(128, 256) + _double_conv(256, 256)
        n += [128 * 4096, 128, 128 * 4096, 128, 4096 * 128, 4096]
        for ci, co in ((256, 128), (128, 64), (64, 64)):
            n += [4 * ci * co, co, co, co]
        return n + [192, 3]
    wide = module == "unet1024"    # VAEUnet1024(image 224, latent 64), 88 tensors; else VAEUnet256(image 32, latent 128), 70 tensors
    c = (64, 128, 256, 512, 1024) if wide else (64, 128, 256, 256)
    latent, features = (64, 200704) if wide else (128, 4096)
    n, ci = [], 3
    for co in c:
        n += _double_conv(ci, co)
        ci = co
    n += [latent * features, latent] * 2 + [features * latent, features]
    ups = (((1024, 512, 1024), (512, 256, 512), (256, 128, 256), (128, 64, 128)) if wide
           else ((256, 128, 384), (128, 64, 192), (64, 64, 128)))
    for ci, co, cat in ups:
        n += [4 * ci * co, co] + _double_conv(cat, co)
    return n + [192, 3]


def sizes(case):
    if case["module"] != "ragged":
        return _module_sizes(case["module"])
    rng = random.Random(case["split"])     # sizes spread over their logarithm, odd ones among them
    w = [math.exp(rng.uniform(0.0, 9.0)) for _ in range(case["tensors"])]
    return [max(1, int(case["elements"] * x / sum(w))) for x in w]


def listed():
    return [
        # smallest: one block of the drafts, where a call's latency is all there is
        {"name": "clip block", "op": "clip", "module": "block", "dtype": "fp32", "shift": 0},
        # a U-Net of the drafts, whose 70 tensors are separate allocations
        {"name": "clip unet256", "op": "clip", "module": "unet256", "dtype": "fp32", "shift": 0},
        # many small odd tensors in bf16, none of them aligned
        {"name": "clip ragged bf16", "op": "clip", "module": "ragged", "tensors": 133, "elements": 9_000_001, "split": 5, "dtype": "bf16", "shift": 1},
        # the largest module
        {"name": "clip unet1024", "op": "clip", "module": "unet1024", "dtype": "fp32", "shift": 0},
        # the same four kinds for the step with 32-bit moments, the headline model among them
        {"name": "adamw block", "op": "adamw", "module": "block", "dtype": "fp32", "shift": 0, "clip": False},
        {"name": "adamw conv32", "op": "adamw", "module": "conv32", "dtype": "fp32", "shift": 0, "clip": True},
        {"name": "adamw ragged bf16", "op": "adamw", "module": "ragged", "tensors": 217, "elements": 20_000_003, "split": 9, "dtype": "bf16", "shift": 1, "clip": True},
        {"name": "adamw unet1024", "op": "adamw", "module": "unet1024", "dtype": "fp32", "shift": 0, "clip": True},
        # and with 8-bit moments
        {"name": "adamw8 block", "op": "adamw8", "module": "block", "dtype": "fp32", "shift": 0, "clip": False},
        {"name": "adamw8 conv32", "op": "adamw8", "module": "conv32", "dtype": "fp32", "shift": 0, "clip": True},
        {"name": "adamw8 ragged bf16", "op": "adamw8", "module": "ragged", "tensors": 150, "elements": 9_000_011, "split": 3, "dtype": "bf16", "shift": 0, "clip": True},
        {"name": "adamw8 unet1024", "op": "adamw8", "module": "unet1024", "dtype": "fp32", "shift": 0, "clip": True},
    ]


def draw(rng):
    case = {"op": rng.choice(("clip", "adamw", "adamw8")), "module": "ragged", "dtype": rng.choice(("fp32", "bf16")),
            "tensors": int(math.exp(rng.uniform(0.0, math.log(300.0)))), "elements": int(math.exp(rng.uniform(math.log(2e3), math.log(6e7)))),
            "split": rng.randrange(1 << 20), "shift": rng.randrange(4)}
    if case["op"] != "clip":
        case["clip"] = rng.random() < 0.7
    return case


def work(case):
    """each input read once, each output written once; moments in 8 bits also come back as bf16 values, bf16 parameters with their
    master values in fp32"""
    n, bf16 = sum(sizes(case)), case["dtype"] == "bf16"
    p = 2 if bf16 else 4
    if case["op"] == "clip":
        return {"bytes": 2 * p * n, "flops": 3 * n}
    moved = 3 * p + (4 + 4 if bf16 else 0)                   # parameter both ways, gradient; remainder both ways, master
    moved += 16 if case["op"] == "adamw" else 2 + 2 + 4      # moments both ways (and their values)
    return {"bytes": moved * n, "flops": (15 if case["op"] == "adamw" else 45) * n}


# ------------------------------------------------------------------------------------------------ inputs
def _layout(case):
    n = sizes(case)
    start, at = [], 0
    for k in n:
        start.append(at)
        at += -(-k // BLOCK) * BLOCK
    return n, start, at


def _arena(total, case, values):
    store = torch.zeros(total + case["shift"], device="cuda", dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    store[case["shift"]:] = values
    return store[case["shift"]:]


def _inputs(case, seed):
    """gradients of a scale that differs from tensor to tensor by a factor of up to 100, one element in 20 exactly zero with zero
    moments; parameters of the scale of an initialised layer; moments of a run some hundred steps old"""
    n, start, total = _layout(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw_ = lambda: torch.randn(total, device="cuda", generator=gen)  # noqa: E731
    count = torch.tensor(n, device="cuda")
    which = torch.repeat_interleave(torch.arange(len(n), device="cuda"), (count + BLOCK - 1) // BLOCK * BLOCK)
    index = (torch.arange(total, device="cuda") - torch.tensor(start, device="cuda")[which]).int()      # within the tensor
    scale = torch.pow(10.0, torch.rand(len(n), device="cuda", generator=gen) * -2.0 - 2.0)[which]
    scale = scale * (index < count[which])
    alive = (torch.rand(total, device="cuda", generator=gen) > 0.05).float() * scale
    s = {"n": n, "start": start, "index": index, "g": _arena(total, case, draw_() * alive)}
    if case["op"] == "clip":
        return s
    master = draw_() * 0.05 * (scale > 0)
    s["m"], s["v"] = draw_() * 0.3 * alive, (draw_().square() + 0.2) * alive.square()
    s["t"] = 300 + seed % 700
    if case["dtype"] == "bf16":
        p, s["remainder"] = _split(master)
        s["p"] = _arena(total, case, p)
    else:
        s["p"] = _arena(total, case, master)
    if case["op"] == "adamw8":
        half = torch.full_like(index, 1 << 19).view(-1, BLOCK)
        s["qm"], s["qv"], s["bm"], s["bv"] = _pack8(s.pop("m").view(-1, BLOCK), s.pop("v").view(-1, BLOCK), half, half)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:      # what a program has before its first step: parameters with gradients, and an optimizer with its state
        from vae_amd.optim import MultiAdamW
        cut = lambda x, k: x[s["start"][k]:s["start"][k] + s["n"][k]]  # noqa: E731
        s["params"] = [torch.nn.Parameter(cut(s["g" if case["op"] == "clip" else "p"], k).clone() if case["op"] == "clip" else cut(s["p"], k)) for k in range(len(s["n"]))]
        for k, p in enumerate(s["params"]):
            p.grad = cut(s["g"], k)
        if case["op"] != "clip":
            s["opt"] = MultiAdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=WEIGHT_DECAY,
                                  state_bits=8 if case["op"] == "adamw8" else 32)
            saved = s["opt"].state_dict()
            for k in range(len(s["n"])):
                e = saved["state"][k] = {"step": s["t"]}
                if case["op"] == "adamw8":
                    rows = slice(s["start"][k] // BLOCK, s["start"][k] // BLOCK + -(-s["n"][k] // BLOCK))
                    e["exp_avg_q"], e["exp_avg_sq_q"] = cut(s["qm"].view(-1), k), cut(s["qv"].view(-1), k)
                    e["exp_avg_base"], e["exp_avg_sq_base"] = s["bm"].view(-1)[rows], s["bv"].view(-1)[rows]
                else:
                    e["exp_avg"], e["exp_avg_sq"] = cut(s["m"], k), cut(s["v"], k)
                if case["dtype"] == "bf16":
                    e["remainder"] = cut(s["remainder"], k)
            s["opt"].load_state_dict(saved)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _split(master):
    """(bf16 parameter, int16 remainder) of an fp32 master: the magnitude bits rounded to their upper half, ties up"""
    bits = master.abs().view(torch.int32)
    hi = (bits + 0x8000) >> 16
    p = (hi << 16).view(torch.float32)
    return torch.where(torch.signbit(master), -p, p).to(torch.bfloat16), (bits - (hi << 16)).to(torch.int16)


def _join(p, remainder):
    p = p.float()
    w = (p.abs().view(torch.int32) + remainder.int()).clamp(min=0).view(torch.float32)
    return torch.where(torch.signbit(p), -w, w)


def _dither(index, step, rate):
    return (((index.long() * A + step * rate) & 0xFFFFFFFF) >> 12).int().view(-1, BLOCK)


def _pack8(m, v, dm, dv):
    """codes and bases of moments in rows of one block"""
    a, minus = m.abs(), (m < 0).int() << 7
    am, av = a.view(torch.int32), v.view(torch.int32)
    top = lambda x: ((x.amax(1, keepdim=True) + 0xFFFFF) >> 20).clamp(max=0x7F7)  # noqa: E731
    bm, bv = (top(am) - 127).clamp(min=0), (top(av) - 254).clamp(min=0)
    cv = (((av + dv) >> 20) - bv).clamp(1, 254) * (v > 0)
    low = ((bm + 1) << 20).view(torch.float32)                               # the smallest level of exp_avg
    cm = torch.where(a >= low, (((am + dm) >> 20) - bm).clamp(max=127), (a > dm.float() * (low * 2.0 ** -20)).int())
    return torch.where(cm > 0, cm + minus, cm).to(torch.uint8), cv.to(torch.uint8), bm, bv


def _unpack8(qm, qv, bm, bv):
    cm, cv = qm.int() & 127, qv.int()
    m = (((bm + cm) << 20) * (cm > 0)).view(torch.float32)
    return torch.where(qm > 127, -m, m), (((bv + cv) << 20) * (cv > 0)).view(torch.float32)


def _norm(g):
    return g.double().square().sum().sqrt()                                  # a long sum: 64 bits


def _coefficient(norm):
    return (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()


def run(s):
    case = s["case"]
    eight, bf16 = case["op"] == "adamw8", case["dtype"] == "bf16"
    if own:
        if case["op"] == "clip":
            from vae_amd.optim import clip_grad_norm_
            return {"norm": clip_grad_norm_(s["params"], MAX_NORM), "grads": s["g"]}
        s["opt"].step(max_norm=MAX_NORM if case["clip"] else None)
        m, v = s["opt"].flat_moments()
        out = {"params": s["p"], "exp_avg": m, "exp_avg_sq": v}
        if bf16:
            out["master"] = s["opt"].flat_master()
        return out
    g = s["g"].float()
    if case["op"] == "clip":
        norm = _norm(g)
        s["g"].copy_(g * _coefficient(norm))
        return {"norm": norm.float(), "grads": s["g"]}
    if case["clip"]:
        g = g * _coefficient(_norm(g))
    s["t"] += 1
    t = s["t"]
    p = _join(s["p"], s["remainder"]) if bf16 else s["p"]
    m, v = _unpack8(s["qm"], s["qv"], s["bm"], s["bv"]) if eight else (s["m"], s["v"])
    m, v = BETA1 * m.view(-1) + (1 - BETA1) * g, BETA2 * v.view(-1) + (1 - BETA2) * g * g
    w = p * (1 - LR * WEIGHT_DECAY)
    w = w - LR / (1 - BETA1 ** t) * m / (v.sqrt() / math.sqrt(1 - BETA2 ** t) + EPS)
    if bf16:
        p, s["remainder"] = _split(w)
        s["p"].copy_(p)
        out = {"params": s["p"], "master": w}
    else:
        s["p"].copy_(w)
        out = {"params": s["p"]}
    if eight:
        s["qm"], s["qv"], s["bm"], s["bv"] = _pack8(m.view(-1, BLOCK), v.view(-1, BLOCK), _dither(s["index"], t, B_M), _dither(s["index"], t, B_V))
        m, v = (x.view(-1).to(torch.bfloat16) for x in _unpack8(s["qm"], s["qv"], s["bm"], s["bv"]))      # 4 significant bits: exact in bf16
    else:
        s["m"], s["v"] = m, v
    return {**out, "exp_avg": m, "exp_avg_sq": v}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """the definition in 64 bits: levels by mantissa and exponent instead of bit patterns"""
    s = _inputs(case, seed)
    g = s["g"].double()
    norm = g.pow(2).sum().sqrt()
    coefficient = min(1.0, MAX_NORM / (float(norm) + 1e-6))
    if case["op"] == "clip":
        return {"norm": norm, "grads": g * coefficient}
    if case["clip"]:
        g = g * coefficient
    t = s["t"] + 1
    p = s["p"].double()
    if case["dtype"] == "bf16":
        # parameter and remainder are the 32 bits of the master's magnitude
        magnitude = (s["p"].float().abs().view(torch.int32) + s["remainder"].int()).view(torch.float32).double()
        p = torch.where(torch.signbit(p), -magnitude, magnitude)
    if case["op"] == "adamw8":
        m, v = _unpack8(s["qm"], s["qv"], s["bm"], s["bv"])
        m, v = m.reshape(-1).double(), v.reshape(-1).double()
    else:
        m, v = s["m"].double(), s["v"].double()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g.pow(2) * (1 - BETA2)
    w = p - LR * WEIGHT_DECAY * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out = {"params": w}
    if case["dtype"] == "bf16":
        fraction, e = torch.frexp(w.abs())                                   # fraction in [1/2, 1): 8 significant bits, ties up
        out = {"params": torch.copysign((fraction * 256 + 0.5).floor() / 256 * torch.exp2(e.double()), w), "master": w}
    if case["op"] == "adamw8":
        m, v = _exact_levels(m, s["index"], t, B_M, 127, True), _exact_levels(v, s["index"], t, B_V, 254, False)
    return {**out, "exp_avg": m, "exp_avg_sq": v}


def _exact_levels(x, index, t, rate, codes, signed):
    x, index = x.view(-1, BLOCK), index.view(-1, BLOCK)
    d = torch.div(torch.remainder(index.long() * A + t * rate, 1 << 32), 1 << 12, rounding_mode="floor").double() / 2 ** 20
    value = lambda level: torch.exp2(torch.div(level, 8, rounding_mode="floor") - 4) * (8 + torch.remainder(level, 8))  # noqa: E731
    fraction, e = torch.frexp(x.abs())
    eighths = fraction * 16                                                  # in [8, 16)
    level = 8 * e.double() + eighths.floor() - 8
    level = torch.where(x == 0, torch.full_like(level, -1e6), level)
    part = eighths - eighths.floor()
    lowest = (level + (part > 0)).amax(1, keepdim=True) - codes + 1          # the largest magnitude, rounded up, has the last code
    rounded = level + (part + d >= 1)
    if signed:
        low = value(lowest.clamp(min=-1000))
        got = torch.where(level >= lowest, value(rounded.clamp(min=-1000)), (x.abs() > d * low) * low)
        got = torch.where(x < 0, -got, got)
    else:
        got = value(torch.maximum(rounded, lowest).clamp(min=-1000))
    return torch.where(x == 0, torch.zeros_like(x), got).view(-1)
