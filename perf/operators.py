"""The operators of a node's local training step, as cases to be measured.

Three operators: a matrix product with bias, residual and activation in its
epilogue (``linear``), group norm with residual and activation over
channels-last images (``group_norm``), and an AdamW step over all tensors of a
model with its two moments held in 32 or in 8 bits (``adamw``).

A case is a dict of plain values. ``run`` computes it by elementary torch
operations in 32 bits where ``own`` is false, and through ``murmura_amd.ops``
where it is true; ``exact`` gives the values in 64 bits.
"""

import math

import torch

own = False

LR, BETAS, EPS, DECAY, SEED = 1e-3, (0.9, 0.999), 1e-8, 0.01, 7
#: steps that an optimizer has done before the measured one
STEPS_DONE = 20
#: consecutive values of the whole parameter vector that share a scale
BLOCK = 256
GN_EPS = 1e-5

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _gn(n, c, h, w, groups, dtype, act, res, train):
    return {"op": "group_norm", "n": n, "c": c, "h": h, "w": w, "groups": groups,
            "dtype": dtype, "act": act, "res": res, "train": train}


def _linear(m, k, n, dtype, act, res, train):
    return {"op": "linear", "m": m, "k": k, "n": n,
            "dtype": dtype, "act": act, "res": res, "train": train}


def _adamw(net, dtype, bits):
    return {"op": "adamw", "net": net, "dtype": dtype, "bits": bits}


def listed():
    cases = {
        # one image through the first norm of a ResNet-18 while a node answers: latency
        "gn one image": _gn(1, 64, 32, 32, 32, "bf16", "relu", False, False),
        # a block's tail, relu(norm(x) + shortcut), at the flagship's batch of 64
        "gn block tail": _gn(64, 64, 32, 32, 32, "bf16", "relu", True, True),
        # a ragged batch of 21x21 maps with channels that fill no vector, in fp32
        "gn ragged fp32": _gn(61, 60, 21, 21, 5, "fp32", "gelu", False, True),
        # large images in large batches: a whole sample is far more than a CU holds
        "gn large images": _gn(128, 256, 56, 56, 32, "bf16", "silu", False, True),
        # the wearables' MLP: a step over a few small tensors: latency
        "adamw small mlp": _adamw("561-256-128-6", "fp32", 32),
        # the flagship CNN in bf16, 62 tensors, moments in 8 bits
        "adamw resnet18 8 bits": _adamw("resnet18", "bf16", 8),
        # the wide MLP of 100M parameters in fp32, moments in 32 bits
        "adamw wide mlp": _adamw("4096-12288-4096-62", "fp32", 32),
        # one row through the wide MLP's first layer: every weight is read for one token
        "linear one row": _linear(1, 4096, 12288, "bf16", "relu", False, False),
        # FEMNIST's first full layer at batch 64: forward and all gradients
        "linear batch 64": _linear(64, 3136, 2048, "bf16", "relu", False, True),
        # a ragged batch of the wearables' 561 features, odd in every direction, in fp32
        "linear ragged fp32": _linear(509, 561, 250, "fp32", "gelu", True, True),
        # the wide MLP's second layer as a residual block's end, many rows at evaluation
        "linear evaluation": _linear(2048, 12288, 4096, "bf16", "gelu", True, False),
        # the wide MLP's first layer over many rows: forward and all gradients
        "linear large": _linear(8192, 4096, 12288, "bf16", "relu", False, True),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    op = rng.choice(("group_norm", "linear", "adamw"))
    dtype = rng.choice(("bf16", "fp32"))
    if op == "group_norm":
        groups, per = rng.choice((1, 2, 3, 4, 5, 8, 16, 32)), _log(rng, 1, 32)
        h = _log(rng, 1, 64)
        w = h if rng.random() < 0.7 else _log(rng, 1, 64)
        # a group of a few values says little of a gradient: all of it cancels
        per = max(per, -(-16 // (h * w)))
        n = _log(rng, 1, 256)
        n = max(1, min(n, 100_000_000 // (groups * per * h * w)))
        return _gn(n, groups * per, h, w, groups, dtype, rng.choice(("none", "relu", "silu", "gelu")),
                   rng.random() < 0.4, rng.random() < 0.7)
    if op == "linear":
        m, k, n = _log(rng, 1, 8192), _log(rng, 8, 8192), _log(rng, 4, 8192)
        return _linear(m, k, n, dtype, rng.choice(("none", "relu", "silu", "gelu")),
                       rng.random() < 0.4, rng.random() < 0.7)
    widths = [_log(rng, 10, 6000) for _ in range(rng.choice((2, 3, 4)))]
    return _adamw("-".join(str(v) for v in widths), dtype, rng.choice((8, 32)))


# ------------------------------------------------------------------ inputs
def _shapes(net):
    """The shapes of a model's parameters, in their order."""
    if net == "resnet18":
        widths = [(64, 64), (64, 64), (64, 128), (128, 128), (128, 256), (256, 256), (256, 512), (512, 512)]
        shapes = [(64, 3, 3, 3), (64,), (64,)]
        for i, o in widths:
            shapes += [(o, 3, 3, i), (o,), (o,), (o, 3, 3, o), (o,), (o,)]
            shapes += [(o, 1, 1, i), (o,), (o,)] if i != o else []
        return shapes + [(10, 512), (10,)]
    widths = [int(v) for v in net.split("-")]
    return [s for i, o in zip(widths, widths[1:]) for s in ((o, i), (o,))]


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "group_norm":
        n, c, h, w = case["n"], case["c"], case["h"], case["w"]

        def image():
            return randn(n, h, w, c).to(dt).permute(0, 3, 1, 2)

        # activations as a convolution leaves them: a level and a spread of each channel's own
        x = (randn(n, h, w, c) * (0.5 + 1.5 * torch.rand(c, generator=gen, device=dev)) + randn(c)).to(dt).permute(0, 3, 1, 2)
        state = {"x": x, "weight": (1 + 0.2 * randn(c)).to(dt), "bias": (0.2 * randn(c)).to(dt),
                 "res": image() if case["res"] else None, "dy": image() if case["train"] else None}
    elif case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        state = {"x": randn(m, k).to(dt), "weight": (randn(n, k) / math.sqrt(k)).to(dt),
                 "bias": (0.2 * randn(n)).to(dt), "res": randn(m, n).to(dt) if case["res"] else None,
                 "dy": randn(m, n).to(dt) if case["train"] else None}
    else:
        shapes = _shapes(case["net"])
        sizes = [math.prod(s) for s in shapes]
        total = sum(sizes)
        flat = (0.05 * randn(total)).to(dt)
        # gradients of different sizes in different tensors; some units are dead
        alive = (torch.rand(total, generator=gen, device=dev) > 0.05).float()
        scale = torch.cat([x.expand(k) for x, k in zip(1e-3 * torch.exp(randn(len(sizes))), sizes)])
        noise = scale * alive
        grads = [g.reshape(s).to(dt) for g, s in zip((noise * randn(total)).split(sizes), shapes)]
        m, v = 0.3 * noise * randn(total), noise.square() * (0.02 + 0.02 * torch.rand(total, generator=gen, device=dev))
        if case["bits"] == 8:
            m, v = _encode(m, True, 1 << 15), _encode(v, False, 1 << 15)
        return {"case": case, "flat": flat, "params": [p.view(s) for p, s in zip(flat.split(sizes), shapes)],
                "grads": grads, "m": m, "v": v,
                "step": torch.full((1,), STEPS_DONE, dtype=torch.int64, device=dev)}
    state["case"] = case
    if case["train"]:
        if case["act"] == "relu":
            # relu has no derivative at its kink: which side a value there takes is
            # the last bit's affair, so what comes back to those places is zero
            z = (_linear_z if case["op"] == "linear" else _group_norm_z)(state)[0].detach()
            state["dy"].masked_fill_(z.abs() < 3e-5 if case["op"] == "linear" else _image(z.abs() < 3e-5, case), 0)
        for key in ("x", "weight", "bias", "res"):
            if state[key] is not None:
                state[key].requires_grad_(True)
    return state


# ------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _through_act(dy, z, act):
    """dy times the activation's derivative at z."""
    if act == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), dy)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return dy * s * (1 + z * (1 - s))
    if act == "gelu":
        return dy * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    return dy


def _linear_z(s):
    """The values before the activation, and what they come from."""
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t() + s["bias"].float()
    return z if s["res"] is None else z + s["res"].float(), x, w


@torch.no_grad()
def _plain_linear(s):
    case, dt = s["case"], s["x"].dtype
    z, x, w = _linear_z(s)
    out = {"y": _act(z, case["act"]).to(dt)}
    if s["dy"] is not None:
        dz = _through_act(s["dy"].float(), z, case["act"])
        out |= {"dx": (dz @ w).to(dt), "dweight": (dz.t() @ x).to(dt), "dbias": dz.sum(0).to(dt)}
        if s["res"] is not None:
            out["dres"] = dz.to(dt)
    return out


def _rows(v, case):
    """[n, pixels, groups, channels of a group], in 32 bits."""
    n, c, h, w, g = (case[k] for k in ("n", "c", "h", "w", "groups"))
    return v.permute(0, 2, 3, 1).reshape(n, h * w, g, c // g).float()


def _image(v, case):
    n, c, h, w = (case[k] for k in ("n", "c", "h", "w"))
    return v.reshape(n, h, w, c).permute(0, 3, 1, 2)


def _group_norm_z(s):
    """The values before the activation, and what they come from."""
    case = s["case"]
    x = _rows(s["x"], case)
    gamma, beta = s["weight"].float().view(x.shape[2:]), s["bias"].float().view(x.shape[2:])
    mean = x.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean((1, 3), keepdim=True) + GN_EPS)
    xhat = (x - mean) * rstd
    z = xhat * gamma + beta
    return z if s["res"] is None else z + _rows(s["res"], case), xhat, rstd, gamma


@torch.no_grad()
def _plain_group_norm(s):
    case, dt = s["case"], s["x"].dtype
    z, xhat, rstd, gamma = _group_norm_z(s)
    out = {"y": _image(_act(z, case["act"]), case).to(dt)}
    if s["dy"] is not None:
        dz = _through_act(_rows(s["dy"], case), z, case["act"])
        d = dz * gamma
        dx = rstd * (d - d.mean((1, 3), keepdim=True) - xhat * (d * xhat).mean((1, 3), keepdim=True))
        out |= {"dx": _image(dx, case).to(dt), "dweight": (dz * xhat).sum((0, 1)).reshape(-1).to(dt),
                "dbias": dz.sum((0, 1)).reshape(-1).to(dt)}
        if s["res"] is not None:
            out["dres"] = _image(dz, case).to(dt)
    return out


def _pow2(e):
    """2**e in 64 bits, e a whole number."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _dither(count, step, device):
    """Three 16-bit numbers for each place of the parameter vector at this step."""
    low = 0xFFFFFFFF
    key = ((SEED * 0x9E3779B1) & low) ^ ((step * 0x85A308D3 + 0x3C6EF372) & low)
    h = (torch.arange(count, dtype=torch.int64, device=device) * 0x9E3779B1 + key) & low
    h = ((h ^ (h >> 16)) * 0x6A09E667) & low
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & low
    h = h ^ (h >> 16)
    return h & 0xFFFF, h >> 16, ((h * 0xA54FF53B) & low) >> 16


def _decode(state, first):
    """The moments that 8-bit codes stand for: 3 bits of mantissa, 4 (first
    moment, with a sign) or 5 (second) of exponent, and a power of two for
    each block. An exponent of zero has no leading one; all bits set are a NaN."""
    codes, exps = state
    top, low = (15, -17) if first else (31, -33)
    c = codes.to(torch.int64)
    mag = c & 127 if first else c
    e, mantissa = mag >> 3, mag & 7
    v = torch.where(e > 0, mantissa + 8, mantissa).double() * _pow2(e.clamp(min=1) - 1 + low)
    v = torch.where(mag == 8 * top + 7, torch.full_like(v, math.nan), v)
    v = torch.where(c > 127, -v, v) if first else v
    scale = _pow2(exps.to(torch.int64) - 126).repeat_interleave(BLOCK)[: codes.numel()]
    return (v * scale).float()


def _encode(x, first, dither):
    """(codes, exponents) of 32-bit values, rounded up where the part that is cut off and the dither carry."""
    top, low = (15, -17) if first else (31, -33)
    a = x.abs()
    finite = torch.where(torch.isfinite(a), a, torch.zeros_like(a))
    padded = torch.nn.functional.pad(finite, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    exps = padded.amax(1).view(torch.int32) >> 23
    scale = _pow2(exps - 126).repeat_interleave(BLOCK)[: x.numel()]
    s = (a.double() / scale).float()
    normal = ((s.view(torch.int32) + (dither << 4) + 8) >> 20) - 8 * (127 - top)
    small = torch.floor(s * 2.0 ** -low + (dither + 0.5) / 65536)
    code = torch.where(s >= 2.0 ** (low + 3), normal.to(torch.int64), small.to(torch.int64))
    if not first:
        code = torch.where(x > 0, code.clamp(min=1), code)
    code = torch.where(torch.isfinite(x), code, torch.full_like(code, 8 * top + 7))
    code = torch.where(torch.signbit(x), code + 128, code) if first else code
    return code.to(torch.uint8), exps.to(torch.uint8)


@torch.no_grad()
def _plain_adamw(s):
    case, flat = s["case"], s["flat"]
    grad = torch.cat([g.reshape(-1) for g in s["grads"]]).float()
    s["step"] += 1
    t = s["step"].double()
    c1, c2 = -torch.expm1(t * math.log(BETAS[0])), -torch.expm1(t * math.log(BETAS[1]))
    eight = case["bits"] == 8
    m = _decode(s["m"], True) if eight else s["m"]
    v = _decode(s["v"], False) if eight else s["v"]
    u_m, u_v, u_p = _dither(flat.numel(), s["step"], flat.device) if eight or case["dtype"] == "bf16" else (None,) * 3
    m = BETAS[0] * m + (1 - BETAS[0]) * grad
    v = BETAS[1] * v + (1 - BETAS[1]) * (grad * grad)
    p = flat.float() * (1 - LR * DECAY) - (LR / c1).float() * (m / (torch.sqrt(v) * (1 / c2.sqrt()).float() + EPS))
    if case["dtype"] == "bf16":  # rounded up with the probability of the part that is cut off
        p = (((p.view(torch.int32) + u_p.to(torch.int32)) >> 16) << 16).view(torch.float32)
    flat.copy_(p)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"params": flat, "exp_avg": s["m"], "exp_avg_sq": s["v"], "step": s["step"]}
    new_m, new_v = _encode(m, True, u_m), _encode(v, False, u_v)
    s["m"][0].copy_(new_m[0])
    s["m"][1].copy_(new_m[1])
    s["v"][0].copy_(new_v[0])
    s["v"][1].copy_(new_v[1])
    # a code has 4 significant bits, so bf16 holds what it stands for as it is
    return {"params": flat, "exp_avg": _decode(s["m"], True).bfloat16(),
            "exp_avg_sq": _decode(s["v"], False).bfloat16(), "step": s["step"]}


# ------------------------------------------------- the framework's operators
def _own_linear(s):
    from murmura_amd import ops

    y = ops.linear_act(s["x"], s["weight"], s["bias"], act=s["case"]["act"], res=s["res"])
    return _own_gradients(s, y)


def _own_group_norm(s):
    from murmura_amd import ops

    y = ops.group_norm_act(s["x"], s["case"]["groups"], s["weight"], s["bias"], eps=GN_EPS,
                           act=s["case"]["act"], res=s["res"])
    return _own_gradients(s, y)


def _own_gradients(s, y):
    if s["dy"] is None:
        return {"y": y}
    leaves = {"dx": s["x"], "dweight": s["weight"], "dbias": s["bias"]}
    if s["res"] is not None:
        leaves["dres"] = s["res"]
    return {"y": y, **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), s["dy"])))}


def _own_adamw(s):
    from murmura_amd import ops

    ops.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], LR, betas=BETAS, eps=EPS,
                   weight_decay=DECAY, seed=SEED)
    m, v = s["m"], s["v"]
    if s["case"]["bits"] == 8:
        m, v = ops.adamw_dequantize(m, v, dtype=torch.bfloat16)
    return {"params": s["flat"], "exp_avg": m, "exp_avg_sq": v, "step": s["step"]}


def run(state):
    op = state["case"]["op"]
    if op == "linear":
        return _own_linear(state) if own else _plain_linear(state)
    if op == "group_norm":
        return _own_group_norm(state) if own else _plain_group_norm(state)
    return _own_adamw(state) if own else _plain_adamw(state)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        xs, ws, ys = m * k, n * k, m * n
        values = xs + ws + n + ys * (2 if case["res"] else 1)
        if case["train"]:
            values += ys * (2 if case["res"] else 1) + xs + ws + n
        return {"bytes": size * values, "flops": (6 if case["train"] else 2) * m * n * k}
    if case["op"] == "group_norm":
        x, c = case["n"] * case["c"] * case["h"] * case["w"], case["c"]
        values = x * (3 if case["res"] else 2) + 2 * c
        if case["train"]:
            values += x * (3 if case["res"] else 2) + 2 * c
        return {"bytes": size * values, "flops": x * (30 if case["train"] else 10)}
    total = sum(math.prod(s) for s in _shapes(case["net"]))
    state = 16 * total if case["bits"] == 32 else 4 * total + 4 * -(-total // BLOCK)
    told = 0 if case["bits"] == 32 else 4 * total  # what the codes stand for, in bf16
    return {"bytes": 3 * size * total + state + told, "flops": 20 * total}


# ------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    leaves = {k: s[k].detach().double().requires_grad_(True) for k in ("x", "weight", "bias", "res") if s[k] is not None}
    f = torch.nn.functional
    if case["op"] == "linear":
        z = f.linear(leaves["x"], leaves["weight"], leaves["bias"])
    else:
        z = f.group_norm(leaves["x"].contiguous(), case["groups"], leaves["weight"], leaves["bias"], GN_EPS)
    if "res" in leaves:
        z = z + leaves["res"]
    act = {"none": lambda v: v, "relu": torch.relu, "silu": f.silu, "gelu": f.gelu}[case["act"]]
    y = act(z)
    if not case["train"]:
        return {"y": y.detach()}
    got = torch.autograd.grad(y, list(leaves.values()), s["dy"].double())
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, got)}}


def _exact_adamw(case, s):
    eight = case["bits"] == 8
    t = STEPS_DONE + 1
    p, g = s["flat"].double(), torch.cat([x.double().reshape(-1) for x in s["grads"]])
    m, v = (_exact_value(s["m"], 15), _exact_value(s["v"], 31)) if eight else (s["m"].double(), s["v"].double())
    m, v = m.lerp(g, 1 - BETAS[0]), v.lerp(g.square(), 1 - BETAS[1])
    p = p - LR * DECAY * p - LR * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
    u_m, u_v, u_p = (u.double() for u in _dither(p.numel(), t, p.device))
    if case["dtype"] == "bf16":
        p = _exact_round(p, 7, u_p / 65536, -133)
    if eight:
        m = _exact_code(m, 15, (u_m + 0.5) / 65536)
        v = torch.maximum(_exact_code(v, 31, (u_v + 0.5) / 65536), (v > 0) * _exact_scale(v) * 2.0 ** -33)
    return {"params": p, "exp_avg": m, "exp_avg_sq": v, "step": None}


def _exact_value(state, top):
    """What 8-bit codes stand for, from a table of all of them."""
    signed = top == 15
    table = []
    for c in range(256):
        e, f = (c & 127 if signed else c) >> 3, (c & 7) / 8
        value = 2.0 ** (e - top) * (1 + f) if e else 2.0 ** (1 - top) * f
        table.append(-value if signed and c > 127 else value)
    table = torch.tensor(table, dtype=torch.float64, device=state[0].device)
    where = torch.arange(state[0].numel(), device=state[0].device) // BLOCK
    return table[state[0].long()] * torch.ldexp(torch.ones_like(table[:1]), state[1].long() - 126)[where]


def _exact_scale(x):
    """The power of two over the largest value of each block, for every value."""
    where = torch.arange(x.numel(), device=x.device) // BLOCK
    most = torch.nn.functional.pad(x.abs(), (0, -x.numel() % BLOCK)).view(-1, BLOCK).amax(1)
    e = torch.where(most > 0, torch.frexp(most).exponent, torch.full_like(most, -126, dtype=torch.int32)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(most), e)[where]


def _exact_round(x, bits, u, least):
    """x on a grid of `bits` bits of mantissa and steps of 2**least at the least, up where the rest and u make one."""
    e = (torch.frexp(x.abs()).exponent - 1 - bits).clamp(min=least)
    unit = torch.ldexp(torch.ones_like(x), e)
    return torch.copysign(torch.floor(x.abs() / unit + u) * unit, x)


def _exact_code(x, top, u):
    scale = _exact_scale(x)
    return _exact_round(x / scale, 3, u, 1 - top - 3) * scale
