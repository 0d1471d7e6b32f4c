"""The operators of the networks that the loss trains, as cases that can be timed and checked.

Three operators, each at the sizes that speech enhancement meets (frames of a
512 point STFT at 16 kHz, hop 256, or samples themselves):

``scan``
    the gated linear recurrence: a training pass (``call`` = ``train``: output,
    final state and every gradient), an evaluation (``infer``: output and final
    state, from a given state) and one frame of running streams (``step``).
``norm``
    the end of a residual block and the start of the next: the branch's gate,
    its norm, the scaled residual, the next block's norm; a training pass or
    an evaluation.
``adamw``
    one AdamW step over all tensors of a network, states in 32 or in 8 bits.

Where ``own`` is false, ``run`` computes them in plain torch operations in 32
bits, rounded once at the end; where it is true it calls the package.
"""

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-pesq_amd"))

own = False

RATE = 8.0  # exponent of the recurrence's decay at an open gate
EPS = 1e-6  # of the norms
LR, BETA1, BETA2, ADAM_EPS, WEIGHT_DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256  # elements that share a scale in 8 bit states
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST_SCAN = 16 * 3751 * 960  # elements of the largest scan in 16 bits
MOST_NORM = 60016 * 1024  # elements of the largest norm with its stream in 32 bits
MOST_WEIGHTS = 48_000_000  # of the largest network in 16 bits


def _scan(name, call, batch, time, channels, dtype, reverse=False, resets=False):
    case = {"kind": "scan", "call": call, "batch": batch, "time": time, "channels": channels, "dtype": dtype,
            "reverse": reverse, "resets": resets}
    return dict(case, name=name) if name else case


def _norm(name, call, rows, channels, dtype, stream, gate=True):
    case = {"kind": "norm", "call": call, "rows": rows, "channels": channels, "dtype": dtype, "stream": stream,
            "gate": gate}
    return dict(case, name=name) if name else case


def _adamw(name, width, blocks, dtype, bits):
    case = {"kind": "adamw", "width": width, "blocks": blocks, "dtype": dtype, "bits": bits}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one frame of one live stream: the smallest call
        _scan("step_1x256_f32", "step", 1, 1, 256, "f32"),
        # one frame of each of 256 live streams on a server
        _scan("step_256x1000_bf16", "step", 256, 1, 1000, "bf16"),
        # the usual training step: 8 clips of 8 s, 501 frames
        _scan("scan_8x501x512_bf16", "train", 8, 501, 512, "bf16"),
        # a minute of 4 recordings enhanced offline, the backward direction of a bidirectional layer
        _scan("scan_4x3751x384_f32_reverse", "infer", 4, 3751, 384, "f32", reverse=True),
        # a recurrence over samples, utterances packed one after another, an odd number of channels
        _scan("scan_1x64000x65_f16_packed", "train", 1, 64000, 65, "f16", resets=True),
        # a full batch of minute long recordings: the largest call
        _scan("scan_16x3751x960_bf16", "train", 16, 3751, 960, "bf16"),
        # one frame of one live stream
        _norm("norm_1x256_f32", "infer", 1, 256, "f32", "f32"),
        # the usual training step: 8 clips of 501 frames
        _norm("norm_4008x512_bf16", "train", 4008, 512, "bf16", "bf16"),
        # a residual stream over the STFT's 257 bins, ungated
        _norm("norm_18537x257_f32_plain", "train", 18537, 257, "f32", "f32", gate=False),
        # a full batch of minute long recordings, the residual stream in 32 bits: the largest call
        _norm("norm_60016x1024_bf16_f32", "train", 60016, 1024, "bf16", "f32"),
        # a small real time enhancer: many short tensors
        _adamw("adamw_256x4_f32", 256, 4, "f32", 32),
        # a large enhancer in bf16 with 8 bit states: the largest call
        _adamw("adamw8_1024x9_bf16", 1024, 9, "bf16", 8),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _channels(rng, channels):
    """Every third width a multiple of 8; joint projections of whole powers of two are left out."""

    channels += rng.choice([0, 0, -channels % 8])
    return channels + (channels in (768, 1024, 3072))


def draw(rng):
    kind = rng.choice(["scan"] * 5 + ["norm"] * 4 + ["adamw"] * 3)
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "scan":
        call = rng.choice(["train", "train", "infer", "step"])
        if call == "step":
            return _scan(None, call, _spread(rng, 1, 256), 1, _spread(rng, 16, 2048), dtype)
        most = MOST_SCAN // (2 if dtype == "f32" else 1)
        channels, batch = _spread(rng, 16, 1536), _spread(rng, 1, 64)
        time = _spread(rng, 1, min(64000, most // (channels * batch)))
        channels = _channels(rng, channels)
        time = min(time, most // (channels * batch))
        return _scan(None, call, batch, time, channels, dtype, rng.random() < 0.4, rng.random() < 0.4)
    if kind == "norm":
        most = MOST_NORM * 2 // 3 if dtype == "f32" else MOST_NORM
        channels = _channels(rng, _spread(rng, 16, 4096))
        rows = _spread(rng, 1, min(240000, most // channels))
        return _norm(None, rng.choice(["train", "train", "infer"]), rows, channels, dtype, rng.choice([dtype, "f32"]),
                     rng.random() < 0.7)
    bits = rng.choice([32, 8])
    width = _channels(rng, _spread(rng, 16, 1024))
    weights = MOST_WEIGHTS * (1.0 if dtype != "f32" and bits == 8 else 0.6)
    most = max(1, int((weights / width - 514) / (5 * width)))
    return _adamw(None, width, _spread(rng, 1, min(40, most)), dtype, bits)


# -- inputs -------------------------------------------------------------------


def _shapes(case):
    """Tensors of an enhancer over 257 bins: in and out layers, and per block two
    norms, the residual scale, the joint projection, the decays, the branch's output."""

    w = case["width"]
    block = [(w,), (w,), (w,), (4 * w, w), (w,), (w, w)]
    return [(w, 257), (257, w)] + block * case["blocks"]


def _places(case):
    """(shape, first element) of each tensor where they lie one after another, each
    from a multiple of BLOCK, and the elements in all."""

    places, at = [], 0
    for shape in _shapes(case):
        places.append((shape, at))
        at += -(-math.prod(shape) // BLOCK) * BLOCK
    return places, at


def _view(flat, place):
    shape, at = place
    return flat[at : at + math.prod(shape)].view(shape)


def _code_scale(blocks):
    """Scale of each block, and its reciprocal (0 for blocks too small to hold)."""

    scale = blocks.abs().amax(1, keepdim=True)
    scale = torch.where(scale < 2.0**-100, torch.zeros_like(scale), scale)
    return scale, torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))


def _codes_m(flat):
    """8 bit codes of the first moment: sign(m) 127 sqrt(|m| / scale)."""

    blocks = flat.view(-1, BLOCK)
    scale, inverse = _code_scale(blocks)
    code = torch.round(torch.sqrt(blocks.abs() * inverse) * 127.0)
    return torch.where(blocks < 0, -code, code).to(torch.int8).view(-1), scale.view(-1)


def _codes_v(flat):
    """8 bit codes of the second moment: 255 (v / scale)^(1/4), 1 at least where v > 0."""

    blocks = flat.view(-1, BLOCK)
    scale, inverse = _code_scale(blocks)
    code = torch.round(torch.sqrt(torch.sqrt(blocks * inverse)) * 255.0)
    code = torch.where((blocks > 0) & (scale > 0), code.clamp(min=1.0), code)
    return code.to(torch.uint8).view(-1), scale.view(-1)


def _values_m(code, scale):
    part = code.float().view(-1, BLOCK) / 127.0
    return (part.abs() * part * scale.view(-1, 1)).view(-1)


def _values_v(code, scale):
    part = code.float().view(-1, BLOCK) / 255.0
    part = part * part
    return (part * part * scale.view(-1, 1)).view(-1)


def _make_adamw(case, seed):
    """Weights, gradients and moments of all tensors, one after another in one
    allocation each (gaps of zeros between them)."""

    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    places, total = _places(case)
    p, grad, m, v = (torch.zeros(total, device="cuda") for _ in range(4))
    for shape, at in places:
        size = 0.02 * torch.rand((), generator=g, device="cuda") + 1e-4
        # gradients over two decades from row to row
        rows = 10 ** (2 * torch.rand(shape[:1] + (1,) * (len(shape) - 1), generator=g, device="cuda") - 2) * size
        noise = [torch.randn(shape, generator=g, device="cuda") for _ in range(4)]
        for flat, values in ((p, noise[0] / math.sqrt(shape[-1])), (grad, noise[1] * rows), (m, noise[2] * rows * 0.3),
                             (v, (noise[3].square() * 0.5 + 0.5) * rows.square())):
            _view(flat, (shape, at)).copy_(values)
    if case["bits"] == 8:
        m, v = _codes_m(m), _codes_v(v)
    return {"case": case, "step": 1000 + seed % 1000, "p": p.to(dtype), "g": grad.to(dtype), "m": m, "v": v}


def _make_scan(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, batch, time, channels = TYPES[case["dtype"]], case["batch"], case["time"], case["channels"]
    shape = (batch, channels) if case["call"] == "step" else (batch, time, channels)
    state = {"case": case}
    # x and the two gates' arguments, side by side as one linear layer leaves them
    joint = torch.randn(shape[:-1] + (3 * channels,), generator=g, device="cuda").to(dtype)
    state["x"], state["r"], state["i"] = joint.split(channels, -1)
    # decays a^RATE at an open gate from 0.9 to 0.999
    slow = 0.9 + 0.099 * torch.rand(channels, generator=g, device="cuda")
    state["decay"] = torch.log(torch.expm1(-torch.log(slow) / RATE))
    state["h0"] = torch.randn(batch, channels, generator=g, device="cuda")
    state["reset"] = None
    if case["resets"]:
        state["reset"] = torch.rand(batch, time, generator=g, device="cuda") < 1.0 / max(2.0, min(time / 4, 4000.0))
    if case["call"] == "train":
        state["g_y"] = torch.randn(shape, generator=g, device="cuda").to(dtype)
        state["g_h"] = torch.randn(batch, channels, generator=g, device="cuda")
        for name in ("x", "r", "i", "decay", "h0"):
            state[name] = state[name].detach().requires_grad_()
    return state


def _make_norm(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, stream = TYPES[case["dtype"]], TYPES[case["stream"]]
    shape = (case["rows"], case["channels"])
    state = {"case": case}
    # frames of very different loudness
    level = 10 ** (2 * torch.rand(shape[0], 1, generator=g, device="cuda") - 1)
    state["x"] = (torch.randn(shape, generator=g, device="cuda") * level).to(stream)
    state["branch"] = (torch.randn(shape, generator=g, device="cuda") * level).to(dtype)
    state["gate"] = torch.randn(shape, generator=g, device="cuda").to(dtype) if case["gate"] else None
    for name, mean in (("post", 1.0), ("scale", 0.3), ("pre", 1.0)):
        state[name] = mean + 0.1 * torch.randn(shape[1], generator=g, device="cuda")
    if case["call"] == "train":
        state["g_x"] = torch.randn(shape, generator=g, device="cuda").to(stream)
        state["g_n"] = torch.randn(shape, generator=g, device="cuda").to(dtype)
        for name in _norm_inputs(case):
            state[name].requires_grad_()
    return state


def _norm_inputs(case):
    return ["x", "branch"] + (["gate"] if case["gate"] else []) + ["post", "scale", "pre"]


def _optimizer(state):
    """The package's optimizer over the state's tensors, in the middle of a training."""

    from torch_pesq.hip_ops.adamw import HipAdamW

    bits = state["case"]["bits"]
    places, _ = _places(state["case"])
    params = [torch.nn.Parameter(_view(state["p"], place)) for place in places]
    opt = HipAdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=WEIGHT_DECAY, state_bits=bits)
    held = opt.state_dict()
    for k, (shape, at) in enumerate(places):
        one = {"step": state["step"]}
        for name, value in (("exp_avg", state["m"]), ("exp_avg_sq", state["v"])):
            if bits == 8:
                one[name] = _view(value[0], (shape, at))
                one[name + "_scale"] = value[1][at // BLOCK : at // BLOCK + -(-math.prod(shape) // BLOCK)]
            else:
                one[name] = _view(value, (shape, at))
        held["state"][k] = one
    opt.load_state_dict(held)
    for p, place in zip(params, places):
        p.grad = _view(state["g"], place)
    return opt


def prepare(case, seed):
    state = {"scan": _make_scan, "norm": _make_norm, "adamw": _make_adamw}[case["kind"]](case, seed)
    if own and case["kind"] == "adamw":
        state["opt"] = _optimizer(state)
    return state


# -- the plain forms ----------------------------------------------------------


def _prefix(a, b):
    """h_t = a_t h_{t-1} + b_t over the second axis, by doubling."""

    k = 1
    while k < a.shape[1]:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _gates(state):
    x, r, i = (state[k].detach().float() for k in ("x", "r", "i"))
    open_r, open_i = torch.sigmoid(r), torch.sigmoid(i)
    u = RATE * torch.log1p(torch.exp(state["decay"].detach())) * open_r
    return x, open_r, open_i, u, torch.exp(-u), torch.sqrt(-torch.expm1(-2.0 * u))


def _plain_step(state):
    x, _, open_i, _, a, s = _gates(state)
    state["h0"] = a * state["h0"] + s * open_i * x
    return {"y": state["h0"].to(state["x"].dtype), "state": state["h0"]}


def _plain_scan(state):
    case = state["case"]
    x, open_r, open_i, u, a, s = _gates(state)
    flip = (lambda t: t.flip(1)) if case["reverse"] else (lambda t: t)
    x, open_r, open_i, u, a, s = (flip(t) for t in (x, open_r, open_i, u, a, s))
    keep = a
    if state["reset"] is not None:
        keep = a * (~flip(state["reset"]))[..., None]
    h0 = state["h0"].detach()
    b = s * open_i * x
    h = _prefix(keep, torch.cat([b[:, :1] + keep[:, :1] * h0[:, None], b[:, 1:]], 1))
    dtype = state["x"].dtype
    out = {"y": flip(h).to(dtype), "state": h[:, -1].clone()}
    if case["call"] == "infer":
        return out
    g = flip(state["g_y"].float())
    g = torch.cat([g[:, :-1], g[:, -1:] + state["g_h"][:, None]], 1)
    back = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
    g = _prefix(back.flip(1), g.flip(1)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    driven = g * open_i * x
    du = torch.where(s > 0, a * a / s, torch.zeros_like(s)) * driven - keep * before * g
    out["g_x"] = flip(g * s * open_i).to(dtype)
    out["g_r"] = flip(du * u * (1.0 - open_r)).to(dtype)
    out["g_i"] = flip(driven * s * (1.0 - open_i)).to(dtype)
    out["g_decay"] = (du * open_r).sum((0, 1)) * RATE * torch.sigmoid(state["decay"].detach())
    out["g_h0"] = keep[:, 0] * g[:, 0]
    return out


def _plain_norm(state):
    case = state["case"]
    names = _norm_inputs(case)
    t = {k: state[k].detach().float().requires_grad_(case["call"] == "train") for k in names}
    y = t["branch"]
    if case["gate"]:
        y = y * (t["gate"] * torch.sigmoid(t["gate"]))
    z = y * torch.rsqrt(y.square().mean(1, keepdim=True) + EPS) * t["post"]
    x = t["x"] + t["scale"] * z
    n = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * t["pre"]
    out = {"x": x.detach().to(state["x"].dtype), "n": n.detach().to(state["branch"].dtype)}
    if case["call"] == "train":
        grads = torch.autograd.grad((x, n), [t[k] for k in names], (state["g_x"].float(), state["g_n"].float()))
        out.update({"g_" + k: v.to(state[k].dtype) for k, v in zip(names, grads)})
    return out


def _plain_adamw(state):
    eight = state["case"]["bits"] == 8
    state["step"] += 1
    step_size = LR / (1.0 - BETA1 ** state["step"])
    correction = 1.0 / math.sqrt(1.0 - BETA2 ** state["step"])
    p, g = state["p"], state["g"].float()
    m, v = (_values_m(*state["m"]), _values_v(*state["v"])) if eight else (state["m"], state["v"])
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    update = m / (torch.sqrt(v) * correction + ADAM_EPS)
    p.copy_(p.float() * (1.0 - LR * WEIGHT_DECAY) - update * step_size)
    if eight:
        state["m"], state["v"] = _codes_m(m), _codes_v(v)
        m, v = _values_m(*state["m"]), _values_v(*state["v"])
    else:
        state["m"], state["v"] = m, v
    return {"p": p, "m": m, "v": v}


# -- a pass -------------------------------------------------------------------


def _own_scan(state):
    from torch_pesq.hip_ops.recurrence import gated_recurrence, gated_recurrence_step

    case = state["case"]
    if case["call"] == "step":
        y = gated_recurrence_step(state["x"], state["r"], state["i"], state["decay"], state["h0"], rate=RATE)
        return {"y": y, "state": state["h0"]}
    y, last = gated_recurrence(state["x"], state["r"], state["i"], state["decay"], initial_state=state["h0"],
                               reset=state["reset"], reverse=case["reverse"], rate=RATE)
    out = {"y": y, "state": last}
    if case["call"] == "train":
        names = ("x", "r", "i", "decay", "h0")
        grads = torch.autograd.grad((y, last), [state[k] for k in names], (state["g_y"], state["g_h"]))
        out.update({"g_" + k: v for k, v in zip(names, grads)})
    return out


def _own_norm(state):
    from torch_pesq.hip_ops.norm import residual_norm

    case = state["case"]
    x, n = residual_norm(state["x"], state["branch"], state["post"], gate=state["gate"], scale=state["scale"],
                         next_weight=state["pre"], eps=EPS)
    out = {"x": x, "n": n}
    if case["call"] == "train":
        names = _norm_inputs(case)
        grads = torch.autograd.grad((x, n), [state[k] for k in names], (state["g_x"], state["g_n"]))
        out.update({"g_" + k: v for k, v in zip(names, grads)})
    return out


def _own_adamw(state):
    state["opt"].step()
    m, v = state["opt"].moments()
    return {"p": state["p"], "m": m, "v": v}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"scan": _own_scan, "norm": _own_norm, "adamw": _own_adamw}[kind](state)
    if kind == "scan":
        return _plain_step(state) if state["case"]["call"] == "step" else _plain_scan(state)
    return {"norm": _plain_norm, "adamw": _plain_adamw}[kind](state)


# -- what a pass cannot do without --------------------------------------------


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["kind"] == "scan":
        values, states = case["batch"] * case["time"] * case["channels"], case["batch"] * case["channels"]
        train = case["call"] == "train"
        # x, two gates, y; in training the gradients of all four too
        moved = values * size * (8 if train else 4) + 4 * states * (4 if train else 2) + 8 * case["channels"]
        return {"bytes": moved, "flops": values * (75 if train else 25)}
    if case["kind"] == "norm":
        values = case["rows"] * case["channels"]
        wide = {"f32": 4, "bf16": 2, "f16": 2}[case["stream"]]
        branch = 2 if case["gate"] else 1
        # x in and out, the branch and its gate, the next block's input; the same of the gradients
        moved = values * (2 * wide + (branch + 1) * size)
        train = case["call"] == "train"
        return {"bytes": moved * (2 if train else 1) + 24 * case["channels"], "flops": values * (60 if train else 20)}
    values = sum(math.prod(shape) for shape in _shapes(case))
    # weights in and out, gradients, moments in and out; 8 bit ones are also returned as values
    held = 16 if case["bits"] == 32 else 4 + 8 + 16 / BLOCK
    return {"bytes": int(values * (3 * size + held)), "flops": values * (15 if case["bits"] == 32 else 40)}


# -- the same in 64 bits ------------------------------------------------------


def _exact_scan(case, seed):
    state = _make_scan(case, seed)
    x, r, i, decay, h0 = (state[k].detach().double() for k in ("x", "r", "i", "decay", "h0"))
    leaves = [t.requires_grad_() for t in (x, r, i, decay)]
    log_a = -RATE * torch.nn.functional.softplus(decay) * torch.sigmoid(r)
    a = torch.exp(log_a)
    b = torch.sqrt((1.0 - a) * (1.0 + a)) * torch.sigmoid(i) * x
    if case["call"] == "step":
        h = (a * h0 + b).detach()
        return {"y": h, "state": h}
    if state["reset"] is not None:
        a = a.masked_fill(state["reset"][..., None], 0.0)
    order = range(case["time"] - 1, -1, -1) if case["reverse"] else range(case["time"])
    y, before = torch.empty_like(b), torch.empty_like(b)
    h = h0
    with torch.no_grad():
        for t in order:
            before[:, t] = h
            h = torch.addcmul(b[:, t], a[:, t], h)
            y[:, t] = h
        out = {"y": y, "state": h}
        if case["call"] == "infer":
            return out
        g_b = state["g_y"].double()
        carry = state["g_h"].double()
        for t in reversed(order):
            g_b[:, t] += carry
            carry = g_b[:, t] * a[:, t]
    grads = torch.autograd.grad((a, b), leaves, (g_b * before, g_b))
    out.update(zip(("g_x", "g_r", "g_i", "g_decay"), grads))
    return dict(out, g_h0=carry)


def _exact_norm(case, seed):
    state = _make_norm(case, seed)
    names = _norm_inputs(case)
    t = {k: state[k].detach().double() for k in names}
    count = case["channels"]
    sig = torch.sigmoid(t["gate"]) if case["gate"] else None
    y = t["branch"] * t["gate"] * sig if case["gate"] else t["branch"]
    inv_y = ((y * y).sum(1, keepdim=True) / count + EPS) ** -0.5
    unit_y = y * inv_y
    x = t["x"] + t["scale"] * t["post"] * unit_y
    inv_x = ((x * x).sum(1, keepdim=True) / count + EPS) ** -0.5
    unit_x = x * inv_x
    out = {"x": x, "n": unit_x * t["pre"]}
    if case["call"] == "infer":
        return out
    g_n = state["g_n"].double()
    along = g_n * t["pre"]
    g_x = state["g_x"].double() + inv_x * (along - unit_x * (along * unit_x).sum(1, keepdim=True) / count)
    along = g_x * t["scale"] * t["post"]
    g_y = inv_y * (along - unit_y * (along * unit_y).sum(1, keepdim=True) / count)
    both = (g_x * unit_y).sum(0)
    out.update(g_x=g_x, g_branch=g_y * t["gate"] * sig if case["gate"] else g_y)
    if case["gate"]:
        out["g_gate"] = g_y * t["branch"] * sig * (1.0 + t["gate"] * (1.0 - sig))
    return dict(out, g_post=both * t["scale"], g_scale=both * t["post"], g_pre=(g_n * unit_x).sum(0))


def _held64(t, signed):
    """What 8 bits hold of a moment: per block of 256 the largest magnitude in 32
    bits, and each element's share of it to the nearest 127th of its square root
    (first moment) or 255th of its fourth root (second)."""

    levels, power = (127.0, 2) if signed else (255.0, 4)
    rows = t.view(-1, BLOCK)
    top = rows.abs().max(1, keepdim=True).values
    code = torch.floor((rows.abs() / top.clamp(min=1e-300)) ** (1.0 / power) * levels + 0.5)
    if not signed:
        code = torch.where(rows > 0, code.clamp(min=1.0), code)
    return (rows.sign() * (code / levels) ** power * top.float().double()).flatten()


def _expand64(code, scale, signed):
    share = code.double() / (127.0 if signed else 255.0)
    share = share * share.abs() if signed else share**4
    return share * scale.double().repeat_interleave(BLOCK)


def _exact_adamw(case, seed):
    state = _make_adamw(case, seed)
    step = state["step"] + 1
    eight = case["bits"] == 8
    p, g = state["p"].double(), state["g"].double()
    m, v = state["m"], state["v"]
    m, v = (_expand64(*m, signed=True), _expand64(*v, signed=False)) if eight else (m.double(), v.double())
    m = m + (1.0 - BETA1) * (g - m)
    v = v + (1.0 - BETA2) * (g**2 - v)
    m_hat, v_hat = m / (1.0 - BETA1**step), v / (1.0 - BETA2**step)
    p = p - LR * (m_hat / (v_hat**0.5 + ADAM_EPS) + WEIGHT_DECAY * p)
    return {"p": p, "m": _held64(m, True) if eight else m, "v": _held64(v, False) if eight else v}


def exact(case, seed):
    return {"scan": _exact_scan, "norm": _exact_norm, "adamw": _exact_adamw}[case["kind"]](case, seed)
