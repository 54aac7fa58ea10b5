"""Torch reference implementations of every hot op (the bit-level oracle).

Each function here is the semantic definition of a HIP kernel in
murmura_amd/ops/hip/ (K1 to K18). The GPU path
must match these within float tolerance; numerics tests compare the HIP kernel
against the fp32 torch implementation of the same op.

All ops operate on flat state vectors [P] or stacked states [m, P]
(see core/flat.py for why).
"""

from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor


# ---------------------------------------------------------------- K1
def weighted_sum(stacked: Tensor, weights: Tensor, out: Optional[Tensor] = None) -> Tensor:
    """out[p] = sum_i weights[i] * stacked[i, p].

    Reference semantics: ``average_states`` (murmura/aggregation/base.py:76-115)
    and the alpha-blends of balance/ubar/sketchguard/evidential_trust.
    """
    w = weights.to(stacked.dtype)
    res = torch.mv(stacked.t(), w) if stacked.dim() == 2 else stacked * w
    if out is not None:
        out.copy_(res)
        return out
    return res


# ---------------------------------------------------------------- K2 (+K12)
def pairwise_sq_dists(stacked: Tensor) -> Tensor:
    """D2[i, j] = ||x_i - x_j||^2 over rows, computed via the Gram matrix so
    each row is read once (reference computes per-pair per-key with .item()
    syncs — murmura/aggregation/base.py:118-135; krum.py:54-62)."""
    x = stacked.float()
    g = x @ x.t()
    sq = g.diagonal()
    d2 = sq.unsqueeze(0) + sq.unsqueeze(1) - 2.0 * g
    return d2.clamp_min_(0.0)


def pairwise_l2(stacked: Tensor) -> Tensor:
    """D[i, j] = ||x_i - x_j||_2."""
    return pairwise_sq_dists(stacked).sqrt_()


def row_norms(stacked: Tensor) -> Tensor:
    """||x_i||_2 per row (K12; reference: balance.py:91-97)."""
    return stacked.float().norm(dim=-1)


def l2_dists_to(own: Tensor, stacked: Tensor) -> Tensor:
    """d[i] = ||stacked[i] - own||_2 (BALANCE/UBAR stage-1 filtering)."""
    return (stacked.float() - own.float().unsqueeze(0)).norm(dim=-1)


# ---------------------------------------------------------------- K3
def krum_scores(d2: Tensor, num_compromised: int) -> Tensor:
    """score_i = sum of the (m - c - 2) smallest squared distances to others.

    The reference sorts plain L2 distances and sums the m-c-2 smallest
    (krum.py:64-71); we keep squared distances (monotone => same argmin and
    same ordering of candidate sets as summing monotone transforms? NO —
    sums of squares differ from sums of norms). For exact parity we take
    sqrt first.
    """
    m = d2.shape[0]
    d = d2.clamp_min(0).sqrt()
    # exclude self-distance (diagonal) by setting it to +inf before topk
    dd = d.clone()
    dd.fill_diagonal_(float("inf"))
    k = max(m - num_compromised - 2, 1)
    k = min(k, m - 1)
    smallest, _ = torch.topk(dd, k, dim=1, largest=False)
    return smallest.sum(dim=1)


def krum_select(d2: Tensor, num_compromised: int) -> Tensor:
    """argmin of krum scores, returned as a 0-dim device tensor (no host sync)."""
    return torch.argmin(krum_scores(d2, num_compromised))


# ---------------------------------------------------------------- K4/K5
def count_sketch(stacked: Tensor, hash_idx: Tensor, signs: Tensor, sketch_size: int) -> Tensor:
    """s[i, h[p]] += sign[p] * stacked[i, p] for each row i
    (reference: np.bincount with weights, sketchguard.py:91-112)."""
    x = stacked.float() if stacked.dim() == 2 else stacked.float().unsqueeze(0)
    m = x.shape[0]
    out = torch.zeros(m, sketch_size, device=x.device, dtype=torch.float32)
    idx = hash_idx.long().unsqueeze(0).expand(m, -1)
    out.scatter_add_(1, idx, x * signs.float())
    return out if stacked.dim() == 2 else out.squeeze(0)


SKETCH_GROUP = 8


def make_sketch_tables(
    model_dim: int, sketch_size: int, seed: int, device: torch.device,
    group: int = SKETCH_GROUP,
) -> Tuple[Tensor, Tensor]:
    """Hash/sign tables from a seeded RNG (reference: sketchguard.py:71-76 uses
    np.random.RandomState; we use torch.Generator — deterministic per seed,
    shared across all ranks by construction).

    MI355X-native table structure: the BIN assignment is constant within each
    aligned ``group`` of 8 consecutive coordinates while SIGNS stay
    per-element. Per-element signs keep every cross term zero-mean, so sketch
    distances remain unbiased; grouping only raises the collision variance of
    coordinate PAIRS inside one group (8/S of coordinates instead of 1/S —
    negligible at S=1000). What it buys: the GPU kernel accumulates each
    group in registers and issues ONE LDS atomic per group per row instead of
    8 — the kernel is atomic-issue-bound (measured ~200G atomics/s), so this
    is the difference between 2.4 and >10 TB/s effective. The CPU reference
    path below and this table layout produce IDENTICAL sketch values.
    Pass ``group=1`` for reference-style fully independent bins."""
    g = torch.Generator().manual_seed(seed)
    if group > 1:
        ngroups = (model_dim + group - 1) // group
        hg = torch.randint(0, sketch_size, (ngroups,), generator=g, dtype=torch.int64)
        hash_idx = hg.repeat_interleave(group)[:model_dim]
    else:
        hash_idx = torch.randint(
            0, sketch_size, (model_dim,), generator=g, dtype=torch.int64
        )
    signs = torch.randint(0, 2, (model_dim,), generator=g, dtype=torch.int64) * 2 - 1
    return hash_idx.to(device), signs.to(device=device, dtype=torch.float32)


# ---------------------------------------------------------------- K6
def sgd_step(flat_params: Tensor, grad: Tensor, lr: float) -> None:
    """p <- p - lr * g, fused across the whole param prefix
    (reference: fresh torch.optim.SGD per round, core/node.py:74-98)."""
    flat_params.add_(grad, alpha=-lr)


# ---------------------------------------------------------------- K7
def ce_loss_acc(logits: Tensor, targets: Tensor) -> Tuple[Tensor, Tensor]:
    """(summed CE loss, correct count) — fused eval epilogue
    (reference: utils/metrics.py:9-47, ubar.py:204-222)."""
    logits = logits.float()
    loss = torch.nn.functional.cross_entropy(logits, targets, reduction="sum")
    correct = (logits.argmax(dim=1) == targets).sum()
    return loss, correct


# ---------------------------------------------------------------- K8
def evidential_stats(
    logits: Tensor, targets: Tensor
) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """Per-batch sums of (vacuity, entropy, strength, correct) from evidential
    logits: alpha = softplus(logits) + 1, S = sum(alpha), vacuity = K/S,
    entropy over p = alpha/S, strength = S
    (reference: core/node.py:150-179; evidential_trust.py:249-287)."""
    logits = logits.float()
    alpha = torch.nn.functional.softplus(logits) + 1.0
    s = alpha.sum(dim=1)
    k = float(logits.shape[1])
    vacuity = k / s
    p = alpha / s.unsqueeze(1)
    entropy = -(p * p.clamp_min(1e-10).log()).sum(dim=1)
    correct = (alpha.argmax(dim=1) == targets).sum()
    return vacuity.sum(), entropy.sum(), s.sum(), correct


# ---------------------------------------------------------------- K10
def gaussian_inject(flat: Tensor, noise_std: float, seed: int, offset: int = 0) -> Tensor:
    """attacked = flat + N(0, noise_std^2), deterministic from (seed, offset)
    (reference: attacks/gaussian.py:79-90). The HIP kernel uses Philox with the
    same (seed, offset) counter scheme; CPU parity is statistical, not bitwise."""
    g = torch.Generator(device=flat.device).manual_seed(seed + offset)
    noise = torch.randn(flat.shape, generator=g, device=flat.device, dtype=torch.float32)
    return flat + noise.to(flat.dtype) * noise_std


# ---------------------------------------------------------------- K11
def scale_inject(flat: Tensor, lam: float) -> Tensor:
    """attacked = lam * flat (reference: attacks/directed.py:79-89)."""
    return flat * lam


# ------------------------------------------------- the local training step
ACTIVATIONS = ("none", "relu", "silu", "gelu")


def check_act(act: str) -> int:
    """The number of an activation's name, as the kernels know it."""
    if act not in ACTIVATIONS:
        raise ValueError(f"unknown activation {act!r}; options: {list(ACTIVATIONS)}")
    return ACTIVATIONS.index(act)


def _activate(z: Tensor, act: str) -> Tensor:
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.7071067811865476))
    return z


def _wide(t: Tensor) -> Tensor:
    return t if t.dtype == torch.float64 else t.float()


# ---------------------------------------------------------------- K16
def check_group_norm_act(x: Tensor, num_groups: int, weight: Optional[Tensor],
                         bias: Optional[Tensor], res: Optional[Tensor]) -> None:
    if x.dim() not in (2, 4):
        raise ValueError(f"group_norm_act: x must be [N, C] or [N, C, H, W], got {tuple(x.shape)}")
    c = x.shape[1]
    if num_groups < 1 or c < 1 or c % num_groups:
        raise ValueError(f"group_norm_act: {num_groups} groups do not divide {c} channels")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.shape != (c,) or p.device != x.device
                              or p.dtype not in (x.dtype, torch.float32)):
            raise ValueError(f"group_norm_act: {name} must be [{c}] on {x.device}, "
                             f"{x.dtype} or fp32")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("group_norm_act: weight and bias must be of one type")
    if res is not None and (res.shape != x.shape or res.device != x.device
                            or res.dtype != x.dtype):
        raise ValueError("group_norm_act: res must have x's shape, type and device")


def group_norm_act(x: Tensor, num_groups: int, weight: Optional[Tensor] = None,
                   bias: Optional[Tensor] = None, eps: float = 1e-5, act: str = "none",
                   res: Optional[Tensor] = None) -> Tensor:
    """y = act((x - mean) / sqrt(var + eps) * weight + bias (+ res)), mean and
    (biased) variance over the pixels and channels of each group, in 32 bits
    and rounded once."""
    check_group_norm_act(x, num_groups, weight, bias, res)
    check_act(act)
    n, c = x.shape[:2]
    z = _wide(x)
    if x.numel():
        g = z.reshape(n, num_groups, -1)
        d = g - g.mean(2, keepdim=True)
        z = (d / torch.sqrt(d.square().mean(2, keepdim=True) + eps)).reshape(x.shape)
    per_channel = (1, c) + (1,) * (x.dim() - 2)
    if weight is not None:
        z = z * _wide(weight).view(per_channel)
    if bias is not None:
        z = z + _wide(bias).view(per_channel)
    if res is not None:
        z = z + _wide(res)
    y = _activate(z, act).to(x.dtype)
    return y.contiguous(memory_format=torch.channels_last) if x.dim() == 4 else y


# ---------------------------------------------------------------- K17
#: a moment: fp32 [P], or (codes [P], exponents [ceil(P/256)]) in uint8
Moment = Union[Tensor, Tuple[Tensor, Tensor]]
ADAMW_BLOCK = 256


def _pow2(e: Tensor) -> Tensor:
    """2**e in 64 bits for whole e, from its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _moment_form(first: bool) -> Tuple[int, float]:
    """(exponent of the code whose mantissa is bare, smallest code's value)."""
    return (15, 2.0 ** -17) if first else (31, 2.0 ** -33)


def adamw_decode(codes: Tensor, exps: Tensor, first: bool) -> Tensor:
    """fp32 values of an 8-bit moment (the format stands at K17's kernel)."""
    top, least = _moment_form(first)
    c = codes.to(torch.int64)
    mag = c & 127 if first else c
    e = mag >> 3
    value = ((mag & 7) + 8 * (e > 0)).double() * least * _pow2((e - 1).clamp_min(0))
    value = value.masked_fill(mag == 8 * top + 7, math.nan)
    if first:
        value = torch.where(c > 127, -value, value)
    scale = _pow2(exps.to(torch.int64) - 126).repeat_interleave(ADAMW_BLOCK)[: codes.numel()]
    return (value * scale).float()


def adamw_encode(x: Tensor, first: bool, dither: Tensor) -> Tuple[Tensor, Tensor]:
    """(codes, exponents) of fp32 values [P]; dither: 16 random bits a value."""
    top = _moment_form(first)[0]
    a = x.abs()
    finite = torch.isfinite(x)
    blocks = torch.nn.functional.pad(a.masked_fill(~finite, 0.0), (0, -x.numel() % ADAMW_BLOCK))
    exps = blocks.view(-1, ADAMW_BLOCK).amax(1).view(torch.int32) >> 23
    # the code's bits are the top bits of a float whose exponent is off by 127 - top; without a
    # leading one, of a denormal float
    shift = _pow2(top - 1 - exps).repeat_interleave(ADAMW_BLOCK)[: x.numel()]
    bits = (a.double() * shift).float().view(torch.int32).to(torch.int64)
    code = (bits + (dither << 4) + 8) >> 20
    if not first:
        code = torch.where(a > 0, code.clamp_min(1), code)
    code = torch.where(finite, code, 8 * top + 7)
    if first:
        code = code + 128 * torch.signbit(x)
    return code.to(torch.uint8), exps.to(torch.uint8)


def adamw_dither(numel: int, seed: int, t: int, device) -> Tuple[Tensor, Tensor, Tensor]:
    """16 random bits for the first moment, the second and the parameter at
    each place, from a hash of (seed, step, place)."""
    low = 0xFFFFFFFF
    key = ((seed & low) * 0x9E3779B1 & low) ^ (((t & low) * 0x85A308D3 + 0x3C6EF372) & low)
    x = (torch.arange(numel, dtype=torch.int64, device=device) & low) * 0x9E3779B1 + key & low
    x = (x ^ x >> 16) * 0x6A09E667 & low
    x = (x ^ x >> 15) * 0xBB67AE85 & low
    x = x ^ x >> 16
    return x & 0xFFFF, x >> 16, (x * 0xA54FF53B & low) >> 16


def as_list(t: Union[Tensor, Sequence[Tensor]]) -> List[Tensor]:
    return [t] if isinstance(t, Tensor) else list(t)


def _in_memory_order(t: Tensor, like: Tensor) -> Tensor:
    """t's values in the order in which ``like`` (without gaps) holds its own."""
    if t.stride() != like.stride():
        t = torch.empty_strided(like.shape, like.stride(), dtype=t.dtype, device=t.device).copy_(t)
    return torch.as_strided(t, (t.numel(),), (1,))


@torch.no_grad()
def adamw_step(params, grads, exp_avg: Moment, exp_avg_sq: Moment, step: Tensor, lr,
               betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               seed: int = 0) -> None:
    """The semantics of K17, in elementary fp32 operations (see ops.adamw_step)."""
    params, grads = as_list(params), as_list(grads)
    if not params or len(params) != len(grads):
        raise RuntimeError("adamw_step: as many gradients as parameters are wanted")
    numel = sum(p.numel() for p in params)
    eight = not isinstance(exp_avg, Tensor)
    if eight != (not isinstance(exp_avg_sq, Tensor)):
        raise RuntimeError("adamw_step: both moments in the same bits")
    for moment in (exp_avg, exp_avg_sq):
        values = moment[0] if eight else moment
        if values.numel() != numel or values.dtype != (torch.uint8 if eight else torch.float32) or (
                eight and moment[1].numel() != -(-numel // ADAMW_BLOCK)):
            raise RuntimeError("adamw_step: a moment must have a value for each parameter")
    for p, g in zip(params, grads):
        if p.shape != g.shape:
            raise RuntimeError("adamw_step: a gradient must have its parameter's shape")
    step += 1
    t = int(step)
    lr = float(lr)
    c1 = lr / -math.expm1(t * math.log(betas[0])) if betas[0] else lr
    c2 = 1 / math.sqrt(-math.expm1(t * math.log(betas[1]))) if betas[1] else 1.0
    g = torch.cat([_in_memory_order(x, p) for p, x in zip(params, grads)]).float()
    p = torch.cat([_in_memory_order(x, x) for x in params])
    m = adamw_decode(*exp_avg, True) if eight else exp_avg
    v = adamw_decode(*exp_avg_sq, False) if eight else exp_avg_sq
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * (g * g)
    # a root in 64 bits rounds to the right one in 32, which the CPU's own need not be
    root = v.double().sqrt().float()
    new = p.float() * (1 - lr * weight_decay) - c1 * (m / (root * c2 + eps))
    u_m, u_v, u_p = adamw_dither(numel, seed, t, p.device)
    if p.dtype == torch.bfloat16:
        bits = new.view(torch.int32).to(torch.int64) & 0xFFFFFFFF
        up = torch.where((bits & 0x7F800000) == 0x7F800000, 0, u_p)
        rounded = ((bits + up) >> 16) << 16
        rounded = torch.where(rounded >= 1 << 31, rounded - (1 << 32), rounded).to(torch.int32)
        new = torch.where(torch.isnan(new), new, rounded.view(torch.float32)).to(p.dtype)
    for x, y in zip(params, new.split([x.numel() for x in params])):
        torch.as_strided(x, (x.numel(),), (1,)).copy_(y)
    if eight:
        for state, value in zip((exp_avg, exp_avg_sq),
                                (adamw_encode(m, True, u_m), adamw_encode(v, False, u_v))):
            state[0].copy_(value[0])
            state[1].copy_(value[1])
    else:
        exp_avg.copy_(m)
        exp_avg_sq.copy_(v)


# ---------------------------------------------------------------- K18
def check_linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor],
                     res: Optional[Tensor]) -> None:
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_act: weight must be [N, K] for x [..., K], got "
                         f"{tuple(weight.shape)} for {tuple(x.shape)}")
    if weight.dtype != x.dtype or weight.device != x.device:
        raise ValueError("linear_act: weight must have x's type and device")
    n = weight.shape[0]
    if bias is not None and (bias.shape != (n,) or bias.device != x.device
                             or bias.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f"linear_act: bias must be [{n}] on {x.device}, {x.dtype} or fp32")
    if res is not None and (res.shape != (*x.shape[:-1], n) or res.dtype != x.dtype
                            or res.device != x.device):
        raise ValueError("linear_act: res must be [..., N], of x's type and device")


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: str = "none",
               res: Optional[Tensor] = None) -> Tensor:
    """y = act(x @ weight.T + bias + res), in 32 bits and rounded once."""
    check_linear_act(x, weight, bias, res)
    check_act(act)
    z = _wide(x) @ _wide(weight).t()
    if bias is not None:
        z = z + _wide(bias)
    if res is not None:
        z = z + _wide(res)
    return _activate(z, act).to(x.dtype)
