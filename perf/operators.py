"""Cases of three training operators: group norm with an activation, AdamW over many tensors, gradient clipping.

Sizes are those of the segmentation network at 512x1024 with 64 base channels, of the 32x32 classification batches, and
generic odd ones.  `run` computes a case in its plain form, or through the framework where `own` is set.
"""
import math
import random

import torch

own = False

ACTS = ("none", "relu", "relu6", "leakyrelu", "gelu", "hswish", "silu")
SLOPE = 0.2                                  # leaky ReLU, the default of the framework's act_layer
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256                                  # elements that share a scale in the 8-bit states; every tensor starts on one
TOP = 448.0                                  # largest finite e4m3 value
DEV = "cuda:0"


def listed():
    def gn(name, **k):
        return {"name": name, "op": "gn", "dtype": "bf16", "train": True, "residual": False, "act": "relu", **k}

    def opt(name, **k):
        return {"name": name, "op": "adamw", "bits": 32, "odd": False, "clip": 0.0, "step": 100, **k}
    return [
        # one small map of one image, as a serving call makes it: launch latency
        gn("gn_infer_tiny", n=1, c=64, h=16, w=16, groups=32, act="silu", train=False),
        # two full-resolution images, evaluation
        gn("gn_infer_seg", n=2, c=64, h=512, w=1024, groups=32, train=False),
        # a classification batch in 32 bits: many small images
        gn("gn_train_cls_f32", n=64, c=64, h=32, w=32, groups=8, dtype="f32"),
        # a deep stage of the segmentation network with the residual block's second input
        gn("gn_train_deep", n=6, c=512, h=64, w=128, groups=32, residual=True),
        # sizes that fill no tile, four channels to a group, an activation that is not piecewise linear
        gn("gn_train_ragged", n=3, c=80, h=77, w=131, groups=20, act="gelu"),
        # the first stage of the segmentation network at batch 6: the largest activation there is
        gn("gn_train_seg", n=6, c=64, h=512, w=1024, groups=32),
        # a head that is trained alone: six small tensors, launch latency
        opt("adamw32_tiny", tensors=6, largest=2304),
        # the segmentation network's 134 tensors, clipped, in 32 bits and in 8
        opt("adamw32_model", tensors=134, largest=9437184, clip=1.0),
        opt("adamw8_model", tensors=134, largest=9437184, clip=1.0, bits=8),
        # a much larger network, where the states' bytes count most
        opt("adamw8_large", tensors=48, largest=1 << 26, bits=8),
        # clipping by itself, for the other optimisers: the network's gradients, and a few odd ones
        {"name": "clip_model", "op": "clip", "tensors": 134, "largest": 9437184, "odd": False, "clip": 1.0},
        {"name": "clip_odd", "op": "clip", "tensors": 37, "largest": 40001, "odd": True, "clip": 0.5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("gn", "gn", "adamw", "adamw", "clip"))
    if kind == "gn":
        dtype = rng.choice(("bf16", "bf16", "f32"))
        groups, per = rng.choice((1, 2, 4, 8, 16, 20, 32)), rng.choice((1, 2, 3, 4, 5, 8, 10, 16, 32))
        c = groups * per
        n, elems = _log(rng, 1, 64), _log(rng, 20000, 1 << 26)
        hw = max(64, elems // (n * c))
        h = max(4, _log(rng, max(4, math.isqrt(hw) // 3), math.isqrt(hw)))
        return {"op": "gn", "dtype": dtype, "train": rng.random() < 0.7, "residual": rng.random() < 0.4,
                "act": rng.choice(ACTS), "n": n, "c": c, "h": h, "w": max(4, hw // h), "groups": groups}
    case = {"op": kind, "tensors": _log(rng, 4, 150), "largest": _log(rng, 300, 1 << 24), "odd": rng.random() < 0.6,
            "clip": rng.choice((0.5, 1.0, 5.0))}
    if kind == "adamw":
        case |= {"bits": rng.choice((32, 8)), "step": rng.choice((0, 1, 9, 1000)), "clip": rng.choice((0.0, 1.0))}
    return case


def _sizes(case):
    """Element counts of a network's tensors: weights that get smaller by a power law, with a short vector after each."""
    r = random.Random(case["tensors"])
    out = []
    for k in range((case["tensors"] + 1) // 2):
        size = max(1, int(case["largest"] / (1 + k) ** 1.2))
        out += [size - size % 2 + 1 if case["odd"] else max(16, size - size % 16), r.choice((16, 19, 32, 64, 128, 256, 512))]
    return out[:case["tensors"]]


def _layout(case):
    """[(offset, size)] of the tensors in one flat buffer, each at a multiple of BLOCK, and the buffer's length."""
    at, out = 0, []
    for s in _sizes(case):
        out.append((at, s))
        at += -(-s // BLOCK) * BLOCK
    return out, at


def work(case):
    if case["op"] == "gn":
        t = case["n"] * case["c"] * case["h"] * case["w"]
        e = 2 if case["dtype"] == "bf16" else 4
        passes = 2 + case["residual"]                                        # x (and the residual) in, y out
        if case["train"]:
            passes += 3 + (2 if case["residual"] and case["act"] != "none" else 0)   # dy, x in, dx out; residual in, its gradient out
        return {"bytes": t * e * passes, "flops": t * (30 if case["train"] else 10)}
    t = sum(_sizes(case))
    if case["op"] == "clip":
        return {"bytes": t * 8, "flops": t * 3}
    # gradient in, parameter in and out, two states in and out (a byte and a 256th of a scale each in 8 bits)
    state = 4.0 if case["bits"] == 32 else 1.0 + 4.0 / BLOCK
    return {"bytes": t * (12 + 4 * state), "flops": t * (20 if case["bits"] == 32 else 60)}


# ------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)
    if case["op"] == "gn":
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        n, c, h, w = case["n"], case["c"], case["h"], case["w"]
        # activations after a convolution: channels of different mean and spread
        x = randn(n, h, w, c) * (0.5 + 1.5 * torch.rand(c, generator=gen, device=DEV)) + randn(c)
        # a gradient that goes along with the activation and the channel, as one of a loss does, and noise
        dy = 0.5 * randn(n, h, w, c) + 0.3 * randn(c) * x + randn(c)
        s = {"case": case, "x": x.to(dtype).permute(0, 3, 1, 2), "dy": dy.to(dtype).permute(0, 3, 1, 2),
             "weight": torch.nn.Parameter(1 + 0.2 * randn(c)), "bias": torch.nn.Parameter(0.3 * randn(c)), "residual": None}
        if case["residual"]:
            s["residual"] = randn(n, h, w, c).to(dtype).permute(0, 3, 1, 2)
        if own:
            from uresnet_amd import nn
            s["norm"] = nn.GroupNorm(case["groups"], c, eps=EPS)
            s["norm"].weight, s["norm"].bias = s["weight"], s["bias"]
        return s
    layout, total = _layout(case)
    starts = torch.tensor([o for o, _ in layout], device=DEV)
    sizes = torch.tensor([z for _, z in layout], device=DEV)
    which = torch.bucketize(torch.arange(total, device=DEV), starts, right=True) - 1
    inside = torch.arange(total, device=DEV) - starts[which] < sizes[which]                 # the rest is padding: zeros
    spread = (10.0 ** (2 * torch.rand(len(layout), generator=gen, device=DEV) - 4))[which] * inside   # gradients of a tensor: 1e-4 .. 1e-2
    flat_p = 0.05 * randn(total) * inside
    flat_g = randn(total) * spread
    s = {"case": case, "layout": layout, "p": flat_p, "g": flat_g, "step": case.get("step", 0)}
    s["params"] = [torch.nn.Parameter(flat_p[o:o + z]) for o, z in layout]
    for p, (o, z) in zip(s["params"], layout):
        p.grad = flat_g[o:o + z]
    if case["op"] == "clip":
        return s
    if case["step"]:
        m = 0.2 * randn(total) * spread
        v = spread.square() * (0.3 + 1.4 * torch.rand(total, generator=gen, device=DEV))
    else:
        m, v = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
    if case["bits"] == 32:
        s["state"] = {"exp_avg": m, "exp_avg_sq": v}
    else:
        mq, ms = _to_e4m3(m, None)
        rq, rs = _to_e4m3(v.sqrt(), _dither(total, 0))
        s["state"] = {"exp_avg": mq, "exp_avg_scale": ms, "exp_avg_sq_root": rq, "exp_avg_sq_root_scale": rs}
    if own:
        from uresnet_amd import train
        opt = train.AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"],
                          max_grad_norm=case["clip"] or None)
        if case["step"]:
            state = {}
            for i, (o, z) in enumerate(layout):
                b = slice(o // BLOCK, -(-(o + z) // BLOCK))
                state[i] = {k: (t[b] if k.endswith("scale") else t[o:o + z]) for k, t in s["state"].items()}
                state[i]["step"] = torch.tensor(float(case["step"]))
            opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
        del s["state"]
        s["opt"] = opt
    return s


# ------------------------------------------------------------------------------ plain forms
def _act(p, act):
    """Activation of a pre-activation held in 64 bits, and its derivative (64 bits: it jumps where the pre-activation is zero)."""
    one = torch.ones_like(p)
    if act == "none":
        return p, one
    if act == "relu":
        return torch.where(p <= 0, 0 * one, p), torch.where(p <= 0, 0 * one, one)
    if act == "relu6":
        return p.clamp(0, 6), torch.where((p > 0) & (p < 6), one, 0 * one)
    if act == "leakyrelu":
        return torch.where(p > 0, p, SLOPE * p), torch.where(p > 0, one, SLOPE * one)
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(p * math.sqrt(0.5)))
        return p * cdf, cdf + p * torch.exp(-0.5 * p * p) * (1 / math.sqrt(2 * math.pi))
    if act == "hswish":
        return p * (p + 3).clamp(0, 6) / 6, torch.where(p <= -3, 0 * one, torch.where(p < 3, (2 * p + 3) / 6, one))
    sig = 1 / (1 + torch.exp(-p))
    return p * sig, sig * (1 + p * (1 - sig))


def _plain_gn(s):
    case, x = s["case"], s["x"]
    n, c, h, w = x.shape
    g, k, dtype = case["groups"], c // case["groups"], x.dtype

    def split(t):
        return t.permute(0, 2, 3, 1).reshape(n, h * w, g, k)

    def whole(t):
        return t.to(dtype).reshape(n, h, w, c).permute(0, 3, 1, 2)
    weight, bias = s["weight"].detach().view(g, k), s["bias"].detach().view(g, k)
    # long sums, and a pre-activation whose sign decides whole terms of the gradients: 64 bits
    xd = split(x).double()
    mean = xd.mean((1, 3), keepdim=True)
    rstd = ((xd - mean).square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    xhat = (xd - mean) * rstd
    del xd
    pre = xhat * weight + bias
    if s["residual"] is not None:
        pre = pre + split(s["residual"])
    y, slope = _act(pre, case["act"])
    del pre
    if not case["train"]:
        return {"y": whole(y)}
    xhat, rstd = xhat.float(), rstd.float()
    d = split(s["dy"]).float() * slope.float()
    out = {"y": whole(y)}
    del y, slope
    s1 = d.sum(1, dtype=torch.float64)                                  # [n][g][k]
    s2 = (d * xhat).sum(1, dtype=torch.float64)
    m = h * w * k
    a = ((s1 * weight).sum(2) / m).float().view(n, 1, g, 1)
    b = ((s2 * weight).sum(2) / m).float().view(n, 1, g, 1)
    out["dx"] = whole(rstd * (d * weight - a - xhat * b))
    out["dweight"], out["dbias"] = s2.sum(0).float().view(c), s1.sum(0).float().view(c)
    if s["residual"] is not None:
        out["dresidual"] = whole(d)
    return out


def _dither(total, step):
    """20 bits for every element from its place and the step count: what the rounding of the second moment's root adds."""
    mask = 0xFFFFFFFF
    h = (torch.arange(total, device=DEV) * 0x9E3779B9 + step * 0xA3D8F1B5) & mask
    h = ((h ^ (h >> 16)) * 0x45D9F3B5) & mask
    h = ((h ^ (h >> 15)) * 0x2C92774D) & mask
    return (h ^ (h >> 16)) & 0xFFFFF


def _to_e4m3(t, dither):
    """(codes, scales) of blocks of 256 values: to the nearest code, or with a dither down or up in proportion."""
    b = t.view(-1, BLOCK)
    top = b.abs().amax(1).clamp_min(2.0 ** -100)
    y = (b * (TOP / top).unsqueeze(1)).clamp(-TOP, TOP).view(-1)
    if dither is not None:
        y = y.double()
        step = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
        y = torch.floor(y / step + dither.double() * 2.0 ** -20) * step
    return y.float().to(torch.float8_e4m3fn), top / TOP


def _from_e4m3(q, scale):
    return (q.float().view(-1, BLOCK) * scale.unsqueeze(1)).view(-1)


def _norm_and_factor(g, limit):
    norm = g.double().square().sum().sqrt().float()
    return norm, torch.clamp(limit / (norm + 1e-6), max=1.0)


def _plain_adamw(s):
    case, st = s["case"], s["state"]
    s["step"] += 1
    t, g, out = s["step"], s["g"], {}
    if case["clip"]:
        out["grad_norm"], factor = _norm_and_factor(g, case["clip"])
        g = g * factor
    small = case["bits"] == 8
    m = _from_e4m3(st["exp_avg"], st["exp_avg_scale"]) if small else st["exp_avg"]
    v = _from_e4m3(st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"]).square() if small else st["exp_avg_sq"]
    m = m + (g - m) * (1 - BETA1)
    v = v * BETA2 + ((1 - BETA2) * g) * g
    root = v.sqrt()
    s["p"].mul_(1 - LR * DECAY)
    s["p"].sub_(LR / (1 - BETA1 ** t) * (m / (root / math.sqrt(1 - BETA2 ** t) + ADAM_EPS)))
    if small:
        st["exp_avg"], st["exp_avg_scale"] = _to_e4m3(m, None)
        st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"] = _to_e4m3(root, _dither(g.numel(), t))
    else:
        st["exp_avg"], st["exp_avg_sq"] = m, v
    return {"p": s["p"], **st, **out}


def _plain_clip(s):
    norm, factor = _norm_and_factor(s["g"], s["case"]["clip"])
    s["g"].mul_(factor)
    return {"grad_norm": norm, "grads": s["g"]}


# ------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if not own:
        with torch.no_grad():
            return {"gn": _plain_gn, "adamw": _plain_adamw, "clip": _plain_clip}[case["op"]](s)
    from uresnet_amd import _lib, ops, train
    if case["op"] == "clip":
        norm = train.clip_grad_norm_(s["params"], case["clip"])
        return {"grad_norm": norm, "grads": s["g"]}
    if case["op"] == "adamw":
        s["opt"].step()
        out = {"p": s["p"], **s["opt"].state_buffers()}
        if case["clip"]:
            out["grad_norm"] = s["opt"].grad_norm
        return out
    code = getattr(_lib, "ACT_" + case["act"].upper())
    if not case["train"]:
        with torch.no_grad():
            return {"y": ops.gn_act(s["x"], s["norm"], residual=s["residual"], act=code, slope=SLOPE)}
    x = s["x"].detach().requires_grad_()
    r = None if s["residual"] is None else s["residual"].detach().requires_grad_()
    y = ops.gn_act(x, s["norm"], residual=r, act=code, slope=SLOPE)
    wrt = [x, s["weight"], s["bias"]] + ([] if r is None else [r])
    return dict(zip(("dx", "dweight", "dbias", "dresidual"), torch.autograd.grad(y, wrt, s["dy"])), y=y.detach())


# ------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gn":
        F = torch.nn.functional
        f = {"none": lambda t: t, "relu": F.relu, "relu6": F.relu6, "leakyrelu": lambda t: F.leaky_relu(t, SLOPE),
             "gelu": F.gelu, "hswish": F.hardswish, "silu": F.silu}[case["act"]]
        names = ["x", "weight", "bias"] + (["residual"] if case["residual"] else [])
        t = {k: s[k].detach().double().contiguous().requires_grad_(case["train"]) for k in names}
        pre = F.group_norm(t["x"], case["groups"], t["weight"], t["bias"], EPS)
        y = f(pre + t["residual"] if case["residual"] else pre)

        def last(v):
            return v.contiguous(memory_format=torch.channels_last) if v.dim() == 4 else v
        if not case["train"]:
            return {"y": last(y)}
        grads = torch.autograd.grad(y, [t[k] for k in names], s["dy"].double().contiguous())
        return {"y": last(y.detach()), **{"d" + k: last(v) for k, v in zip(names, grads)}}
    g = s["g"].double()
    out = {}
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        out["grad_norm"] = norm
        g = g * min(1.0, case["clip"] / (norm.item() + 1e-6))
    if case["op"] == "clip":
        return {"grads": g, **out}
    codes = torch.arange(127, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn).double()     # 0 .. 448

    def value(q, scale):
        return q.double() * scale.double().repeat_interleave(BLOCK)

    def quantise(t, u):
        scale = t.view(-1, BLOCK).abs().amax(1).clamp_min(2.0 ** -100) / TOP
        a = (t / scale.repeat_interleave(BLOCK)).abs().clamp_max(TOP)
        lo = (torch.bucketize(a, codes, right=True) - 1).clamp(0, 125)
        part = (a - codes[lo]) / (codes[lo + 1] - codes[lo])
        up = torch.where(lo % 2 == 0, part > 0.5, part >= 0.5) if u is None else part + u.double() / 2.0 ** 20 >= 1
        return codes[lo + up.long()] * t.sign(), scale
    st, t = s["state"], case["step"] + 1
    if case["bits"] == 8:
        m, v = value(st["exp_avg"], st["exp_avg_scale"]), value(st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"]) ** 2
    else:
        m, v = st["exp_avg"].double(), st["exp_avg_sq"].double()
    m, v = BETA1 * m + (1 - BETA1) * g, BETA2 * v + (1 - BETA2) * g * g
    denom = (v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS
    p = s["p"].double()
    out["p"] = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / denom
    if case["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    out["exp_avg"], out["exp_avg_scale"] = quantise(m, None)
    out["exp_avg_sq_root"], out["exp_avg_sq_root_scale"] = quantise(v.sqrt(), _dither(m.numel(), t))
    return out
