"""Measured cases of the layer-normalisation and weight-update operators: what they compute in plain torch operations, and the
calls that a user of `downscaling.engine.hipops.HipOps` makes for the same work.

Three operators:
  layernorm_fwd / layernorm_bwd   normalisation over the last axis of [rows, C] tensors, and its three gradients;
  adamw, states in 32 bits        one step over a list of tensors, optionally with the gradients clipped by their global norm
                                  and a 16-bit copy of the weights written beside the 32-bit ones;
  adamw, states in 8 bits         the same with both moments held as one byte per element and one scale per 256 elements.
"""
import math
import os
import random
import sys

import torch

own = False          # False: the plain forms below; True: the framework's operators

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
LN_EPS = 1e-3        # the framework's LayerNormalization
BLOCK = 256          # elements that share a scale of the 8-bit moments; every tensor's state starts at a whole block
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM, STEPS_DONE = 1e-4, 0.9, 0.999, 1e-8, 0.01, 1.0, 40

# (elements, takes weight decay) of the discriminator's 32 trainable variables at 256 x 256 and of the generator's 25
DISCRIMINATOR = [(144, 1), (144, 1), (8, 0), (2880, 1), (9216, 1), (64, 0), (288, 1), (16, 0), (2304, 1), (16, 0), (16, 0), (16, 0),
                 (16, 0), (16, 0), (100352, 1), (64, 0), (64, 0), (64, 0), (401408, 1), (128, 0), (128, 0), (128, 0), (1605632, 1),
                 (256, 0), (256, 0), (256, 0), (6422528, 1), (512, 0), (512, 0), (512, 0), (2048, 1), (1, 0)]
GENERATOR = [(188416, 1), (128, 0), (128, 0), (128, 0), (262144, 1), (128, 0), (128, 0), (128, 0), (589824, 1), (589824, 1), (512, 0),
             (73728, 1), (64, 0), (64, 0), (64, 0), (24576, 1), (32, 0), (32, 0), (32, 0), (64000, 1), (16, 0), (16, 0), (16, 0),
             (288, 1), (2, 0)]
CONVLSTMS = [(144, 1), (144, 1), (8, 0), (2880, 1), (9216, 1), (64, 0)]      # the discriminator's two recurrent layers alone


def tensor_list(case):
    named = {"discriminator": DISCRIMINATOR, "generator": GENERATOR, "convlstms": CONVLSTMS}
    if case["tensors"] in named:
        return named[case["tensors"]]
    r = random.Random(case["split"])           # `count` tensors of uneven sizes, `total` elements together
    w = [math.exp(r.uniform(0.0, 5.0)) for _ in range(case["count"])]
    sizes = [max(1, int(case["total"] * x / sum(w))) for x in w]
    return [(n, int(i % 3 != 2)) for i, n in enumerate(sizes)]


def listed():
    return [
        # one token through a norm: launch latency alone
        {"name": "ln_fwd one row", "op": "ln_fwd", "rows": 1, "C": 1024, "type": "fp32", "pad": 0},
        # a long batch of wide rows in the 16-bit training format
        {"name": "ln_fwd wide bf16", "op": "ln_fwd", "rows": 16384, "C": 4096, "type": "bf16", "pad": 0},
        # odd width inside a wider buffer: rows start at odd addresses
        {"name": "ln_fwd odd fp16", "op": "ln_fwd", "rows": 1537, "C": 5003, "type": "fp16", "pad": 8},
        # the discriminator's full-resolution norm: batch 32, 256 x 256 pixels of 16 channels
        {"name": "ln_bwd maps fp32", "op": "ln_bwd", "rows": 2097152, "C": 16, "type": "fp32", "pad": 0},
        {"name": "ln_bwd wide bf16", "op": "ln_bwd", "rows": 16384, "C": 4096, "type": "bf16", "pad": 0},
        # a short, odd batch
        {"name": "ln_bwd odd fp16", "op": "ln_bwd", "rows": 197, "C": 1155, "type": "fp16", "pad": 5},
        # the discriminator's whole update, clipped
        {"name": "adamw discriminator", "op": "adamw", "bits": 32, "tensors": "discriminator", "p": "fp32", "g": "fp32", "copy": "", "clip": True, "shift": 0},
        # two small layers: latency, and tensors that are aligned to nothing but their type
        {"name": "adamw convlstms", "op": "adamw", "bits": 32, "tensors": "convlstms", "p": "fp32", "g": "fp32", "copy": "", "clip": False, "shift": 1},
        # mixed precision at size: 32-bit master weights, bf16 gradients, the bf16 weights written in the same pass
        {"name": "adamw mixed bf16", "op": "adamw", "bits": 32, "tensors": "split", "count": 24, "total": 64000000, "split": 3, "p": "fp32", "g": "bf16", "copy": "bf16", "clip": True, "shift": 0},
        {"name": "adamw8 discriminator", "op": "adamw", "bits": 8, "tensors": "discriminator", "p": "fp32", "g": "fp32", "copy": "", "clip": False, "shift": 0},
        {"name": "adamw8 generator fp16", "op": "adamw", "bits": 8, "tensors": "generator", "p": "fp32", "g": "fp16", "copy": "fp16", "clip": True, "shift": 0},
        {"name": "adamw8 mixed bf16", "op": "adamw", "bits": 8, "tensors": "split", "count": 37, "total": 128000000, "split": 5, "p": "fp32", "g": "bf16", "copy": "bf16", "clip": True, "shift": 0},
    ]


def draw(rng):
    between = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))      # noqa: E731
    op = rng.choice(["ln_fwd", "ln_bwd", "adamw32", "adamw8"])
    if op.startswith("ln"):
        C = between(8, 16384)
        most = min(2 ** 21, 2 ** 26 // C)
        return {"op": op, "rows": between(1, most), "C": C, "type": rng.choice(sorted(TYPES)), "pad": rng.choice([0, 0, 8, rng.randint(1, 67)])}
    kinds = rng.choice([("fp32", "fp32", ""), ("fp32", "bf16", "bf16"), ("fp32", "fp16", "fp16"), ("fp32", "fp32", "bf16"), ("bf16", "bf16", ""), ("fp16", "fp16", "")])
    return {"op": "adamw", "bits": 8 if op == "adamw8" else 32, "tensors": "split", "count": between(1, 60), "total": between(200, 100000000),
            "split": rng.randint(1, 1 << 20), "p": kinds[0], "g": kinds[1], "copy": kinds[2], "clip": rng.random() < 0.5, "shift": rng.choice([0, 0, 1, 2])}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")      # noqa: E731
    ops = _ops() if own else None
    if case["op"] != "adamw":
        return _prepare_ln(case, normal, ops)
    return _prepare_adamw(case, normal, ops)


def _prepare_ln(case, normal, ops):
    rows, C, t = case["rows"], case["C"], TYPES[case["type"]]
    ld = C + case["pad"]
    view = lambda buf: buf[:, :C]      # noqa: E731
    s = {"op": case["op"], "ops": ops, "gamma": 1 + 0.2 * normal(C), "beta": 0.2 * normal(C)}
    # activations: every channel with a scale and an offset of its own
    x = normal(rows, ld) * torch.exp(0.5 * normal(ld)) + 0.5 * normal(ld)
    s["x"] = view(x.to(t))
    if case["op"] == "ln_fwd":
        s["z"] = view(torch.empty(rows, ld, device="cuda", dtype=t))
        s["mean_rstd"] = torch.empty(rows, 2, device="cuda")
        return s
    x64 = s["x"].double()
    s["mean_rstd"] = torch.stack([x64.mean(1), torch.rsqrt(x64.var(1, unbiased=False) + LN_EPS)], 1).float()      # kept by the forward pass
    s["dz"] = view((normal(rows, ld) * torch.exp(normal(rows, 1))).to(t))
    s["dx"] = view(torch.empty(rows, ld, device="cuda", dtype=t))
    s["dgamma"], s["dbeta"] = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
    return s


def _prepare_adamw(case, normal, ops):
    tensors = tensor_list(case)
    sizes = [n for n, _ in tensors]
    blocks = [-(-n // BLOCK) for n in sizes]
    start = [0]
    for b in blocks:
        start.append(start[-1] + b * BLOCK)
    total, shift = start[-1], case["shift"]
    real = torch.zeros(total, device="cuda")                  # 1 on the tensors' elements, 0 on what fills their last block
    scale = torch.zeros(total // BLOCK, 1, device="cuda")
    decay = torch.zeros(total // BLOCK, 1, device="cuda")
    r = random.Random(len(sizes))
    for n, (a, b), (_, d) in zip(sizes, zip(start, start[1:]), tensors):
        real[a:a + n] = 1
        scale[a // BLOCK:b // BLOCK] = math.exp(r.uniform(-2, 1))
        decay[a // BLOCK:b // BLOCK] = d

    def laid(values, kind):
        buf = torch.zeros(total + shift, device="cuda", dtype=TYPES[kind])
        buf[shift:] = (values * real).to(TYPES[kind])
        return buf[shift:]

    spread = lambda: scale * torch.exp(0.5 * normal(total // BLOCK, BLOCK))      # noqa: E731
    size = 1e-3 * spread()                                    # the usual size of each element's gradient
    s = {"op": "adamw", "ops": ops, "bits": case["bits"], "clip": case["clip"], "t": STEPS_DONE, "decay": decay}
    s["p"] = laid((0.05 * normal(total)), case["p"])
    s["g"] = laid((size * normal(total // BLOCK, BLOCK)).view(-1), case["g"])
    s["copy"] = laid(s["p"].float(), case["copy"]) if case["copy"] else None
    m = (0.3 * size * normal(total // BLOCK, BLOCK)).view(-1) * real
    v = (0.04 * size.square() * torch.exp(0.5 * normal(total // BLOCK, BLOCK))).view(-1) * real
    if case["bits"] == 8:
        (s["m"], s["m_scale"]), (s["v"], s["v_scale"]) = _encode_m(m.view(-1, BLOCK)), _encode_v(v.view(-1, BLOCK))
        s["m_values"], s["v_values"] = (torch.empty(total, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    else:
        s["m"], s["v"], s["m_scale"], s["v_scale"] = m, v, None, None
    s["norm"] = torch.zeros(1, device="cuda") if case["clip"] else None
    if ops is not None:
        cut = lambda buf: [None] * len(sizes) if buf is None else [buf[a:a + n] for a, n in zip(start, sizes)]      # noqa: E731
        entries = [(p, g, float(d), c) for p, g, (_, d), c in zip(cut(s["p"]), cut(s["g"]), tensors, cut(s["copy"]))]
        state = (s["m"], s["v"]) if case["bits"] == 32 else (s["m"], s["v"], s["m_scale"], s["v_scale"])
        s["batch"] = ops.make_adamw(entries, state_bits=case["bits"], state=state)
    return s


def run(s):
    if s["op"] == "ln_fwd":
        return _own_ln_fwd(s) if own else _plain_ln_fwd(s)
    if s["op"] == "ln_bwd":
        return _own_ln_bwd(s) if own else _plain_ln_bwd(s)
    s["t"] += 1
    return _own_adamw(s) if own else _plain_adamw(s)


# ---- the framework's operators --------------------------------------------------------------------------------------------
_loaded = []


def _ops():
    if not _loaded:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wind-downscaling-gan_amd")
        if package not in sys.path:
            sys.path.insert(1, package)
        from downscaling.engine.hipops import HipOps
        _loaded.append(HipOps("cuda:0"))
    return _loaded[0]


def _own_ln_fwd(s):
    s["ops"].layernorm_fwd(s["x"], s["gamma"], s["beta"], LN_EPS, s["z"], s["mean_rstd"])
    return {"z": s["z"], "mean_rstd": s["mean_rstd"]}


def _own_ln_bwd(s):
    s["ops"].layernorm_bwd(s["dz"], s["x"], s["mean_rstd"], s["gamma"], s["dx"], s["dgamma"], s["dbeta"], accumulate=False)
    return {"dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}


def _own_adamw(s):
    s["batch"].step(s["t"], LR, BETA1, BETA2, EPS, DECAY, max_norm=MAX_NORM if s["clip"] else None, norm=s["norm"])
    if s["bits"] == 8:
        s["batch"].moments(s["m_values"], s["v_values"])
        return {"p": s["p"], "copy": s["copy"], "m": s["m_values"], "v": s["v_values"], "norm": s["norm"]}
    return {"p": s["p"], "copy": s["copy"], "m": s["m"], "v": s["v"], "norm": s["norm"]}


# ---- the plain forms ------------------------------------------------------------------------------------------------------
def _plain_ln_fwd(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + LN_EPS)
    return {"z": (d * rstd * s["gamma"] + s["beta"]).to(s["x"].dtype), "mean_rstd": torch.cat([mean, rstd], 1)}


def _plain_ln_bwd(s):
    x, dz = s["x"].float(), s["dz"].float()
    mean, rstd = s["mean_rstd"][:, :1], s["mean_rstd"][:, 1:]
    xh = (x - mean) * rstd
    a = dz * s["gamma"]
    dx = rstd * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dz * xh).sum(0), "dbeta": dz.sum(0)}


def _encode_m(m):
    """(codes, scales) of [blocks, 256] first moments: scale * (q / 127) |q / 127|, the scale the block's largest magnitude."""
    scale = m.abs().amax(1)
    q = torch.round(127 * torch.sqrt(m.abs() / torch.where(scale > 0, scale, 1)[:, None]))
    return (q * torch.sign(m)).to(torch.int8).view(-1), scale


def _encode_v(v):
    """... of second moments: scale * (q / 255)^4; a value above zero keeps a code above zero."""
    scale = v.amax(1)
    q = torch.round(255 * torch.sqrt(torch.sqrt(v / torch.where(scale > 0, scale, 1)[:, None])))
    return torch.where(v > 0, q.clamp(min=1), 0).to(torch.uint8).view(-1), scale


def _decode_m(codes, scale):
    q = codes.view(-1, BLOCK).float() / 127
    return q * q.abs() * scale[:, None]


def _decode_v(codes, scale):
    q = codes.view(-1, BLOCK).float() / 255
    return q * q * (q * q) * scale[:, None]


def _plain_adamw(s):
    p, g, out = s["p"].float().view(-1, BLOCK), s["g"].float().view(-1, BLOCK), {}
    if s["clip"]:
        norm = torch.sqrt((s["g"].double() ** 2).sum()).float()
        g = g * (MAX_NORM / torch.clamp(norm, min=MAX_NORM))
        s["norm"][0] = norm
    if s["bits"] == 8:
        m, v = _decode_m(s["m"], s["m_scale"]), _decode_v(s["v"], s["v_scale"])
    else:
        m, v = s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK)
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    t = s["t"]
    p = p * (1 - LR * DECAY * s["decay"]) - LR / (1 - BETA1 ** t) * m / (torch.sqrt(v) / math.sqrt(1 - BETA2 ** t) + EPS)
    s["p"].copy_(p.view(-1))
    if s["copy"] is not None:
        s["copy"].copy_(p.view(-1))
    if s["bits"] == 8:
        (mq, ms), (vq, vs) = _encode_m(m), _encode_v(v)
        for name, new in (("m", mq), ("m_scale", ms), ("v", vq), ("v_scale", vs)):
            s[name].copy_(new)
        s["m_values"].copy_(_decode_m(mq, ms).view(-1))
        s["v_values"].copy_(_decode_v(vq, vs).view(-1))
        out = {"m": s["m_values"], "v": s["v_values"]}
    else:
        s["m"].copy_(m.view(-1))
        s["v"].copy_(v.view(-1))
        out = {"m": s["m"], "v": s["v"]}
    return {"p": s["p"], "copy": s["copy"], "norm": s["norm"], **out}


def work(case):
    if case["op"] != "adamw":
        n, b, C = case["rows"] * case["C"], BYTES[case["type"]], case["C"]
        if case["op"] == "ln_fwd":
            return {"bytes": 2 * n * b + 8 * C + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": 3 * n * b + 12 * C + 8 * case["rows"], "flops": 15 * n}
    n = sum(k for k, _ in tensor_list(case))
    each = 2 * BYTES[case["p"]] + BYTES[case["g"]] + (BYTES[case["copy"]] if case["copy"] else 0)
    # the moments: read and written as they are held; 8-bit ones come back as values of 16 bits too, scales are 16 bytes per block
    each += 16 if case["bits"] == 32 else 2 + 2 + 4 + 16 / BLOCK
    return {"bytes": n * each, "flops": (20 if case["bits"] == 32 else 40) * n}


# ---- the definitions in 64 bits, for the inputs that prepare() makes -----------------------------------------------------------
def exact(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")      # noqa: E731
    f8 = torch.float64
    if case["op"] != "adamw":
        s = _prepare_ln(case, normal, None)
        x, C = s["x"].to(f8), case["C"]
        if case["op"] == "ln_fwd":
            mean = x.sum(1) / C
            var = (x - mean[:, None]).pow(2).sum(1) / C
            rstd = (var + LN_EPS).pow(-0.5)
            z = torch.addcmul(s["beta"].to(f8), (x - mean[:, None]) * rstd[:, None], s["gamma"].to(f8))
            return {"z": z, "mean_rstd": torch.stack((mean, rstd), dim=1)}
        dz, mean, rstd = s["dz"].to(f8), s["mean_rstd"][:, 0].to(f8), s["mean_rstd"][:, 1].to(f8)
        unit = (x - mean.unsqueeze(1)).mul_(rstd.unsqueeze(1))
        up = dz * s["gamma"].to(f8)
        first, second = up.sum(1) / C, (up * unit).sum(1) / C
        dx = (up - first.unsqueeze(1) - unit * second.unsqueeze(1)) * rstd.unsqueeze(1)
        return {"dx": dx, "dgamma": torch.sum(dz * unit, 0), "dbeta": torch.sum(dz, 0)}
    s = _prepare_adamw(case, normal, None)
    t, held = STEPS_DONE + 1, s["p"].numel() // BLOCK
    per_block = lambda v: v.to(f8).repeat_interleave(BLOCK)      # noqa: E731
    if case["bits"] == 8:
        code = s["m"].to(f8)
        m = per_block(s["m_scale"]) * code.sign() * (code / 127.0).pow(2)
        v = per_block(s["v_scale"]) * (s["v"].to(f8) / 255.0).pow(4)
    else:
        m, v = s["m"].to(f8), s["v"].to(f8)
    g, norm = s["g"].to(f8), None
    if case["clip"]:
        norm = g.pow(2).sum().sqrt()
        if norm > MAX_NORM:
            g = g * (MAX_NORM / norm)
        norm = norm.reshape(1)
    m = m + (1.0 - BETA1) * (g - m)
    v = v + (1.0 - BETA2) * (g.pow(2) - v)
    weights = s["p"].to(f8)
    step = (m / (1.0 - BETA1 ** t)) / ((v / (1.0 - BETA2 ** t)).sqrt() + EPS)
    weights = weights - LR * (step + DECAY * per_block(s["decay"][:, 0]) * weights)
    del step, g
    if case["bits"] == 8:
        top = m.abs().view(held, BLOCK).max(1).values
        part = m.abs() / per_block(top.where(top > 0, torch.ones_like(top)))
        m = m.sign() * ((part.pow(0.5) * 127.0).round() / 127.0).pow(2) * per_block(top)
        top = v.view(held, BLOCK).max(1).values
        part = v / per_block(top.where(top > 0, torch.ones_like(top)))
        v = ((part.pow(0.25) * 255.0).round().clamp(min=1.0) / 255.0).pow(4) * per_block(top) * (v > 0)
    return {"p": weights, "copy": weights if case["copy"] else None, "m": m, "v": v, "norm": norm}
