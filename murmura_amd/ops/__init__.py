"""Op dispatch: hand-written CDNA4 HIP kernels on GPU, torch reference on CPU.

Policy: when a tensor is on a ROCm device the native
extension MUST be present and is always used — a silent eager fallback there
is a bug, so we raise instead. The torch implementations in
``reference.py`` serve the CPU simulation backend and the numerics tests.

Set MURMURA_DISABLE_NATIVE=1 to force the torch path everywhere (debug only).
"""

from __future__ import annotations

import os
from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from murmura_amd.ops import reference as ref

_EXT = None
_EXT_ERR: Optional[str] = None


def _load_ext():
    global _EXT, _EXT_ERR
    if _EXT is not None or _EXT_ERR is not None:
        return _EXT
    try:
        from murmura_amd.ops import _hip_loader

        _EXT = _hip_loader.load()
    except Exception as e:  # noqa: BLE001
        _EXT_ERR = f"{type(e).__name__}: {e}"
        _EXT = None
    return _EXT


def native_available() -> bool:
    return _load_ext() is not None


def _use_native(t: Tensor) -> bool:
    if not t.is_cuda:
        return False
    if os.environ.get("MURMURA_DISABLE_NATIVE") == "1":
        return False
    ext = _load_ext()
    if ext is None:
        raise RuntimeError(
            "murmura_amd HIP extension is required for GPU tensors but failed to "
            f"load: {_EXT_ERR}. Build it with `python -m murmura_amd.ops.build` "
            "(or __graft_entry__.build())."
        )
    return True


# ------------------------------------------------------------------ K1
def weighted_sum(stacked: Tensor, weights: Tensor, out: Optional[Tensor] = None) -> Tensor:
    if _use_native(stacked):
        return _EXT.weighted_sum(stacked, weights.to(stacked.device), out)
    return ref.weighted_sum(stacked, weights, out)


# ------------------------------------------------------------------ K2/K12
def pairwise_sq_dists(stacked: Tensor) -> Tensor:
    if _use_native(stacked):
        return _EXT.pairwise_sq_dists(stacked)
    return ref.pairwise_sq_dists(stacked)


def pairwise_l2(stacked: Tensor) -> Tensor:
    return pairwise_sq_dists(stacked).clamp_min(0).sqrt()


def gram(x: Tensor) -> Tensor:
    """Full [m, m] Gram matrix; accepts chunked column views (stride(0) > n)
    so exchange can accumulate it chunk-by-chunk while later chunks are still
    on the wire."""
    if _use_native(x):
        xx = x if x.stride(1) == 1 else x.contiguous()
        return _EXT.gram(xx)
    xf = x.float()
    return xf @ xf.t()


def sq_dists_from_gram(g: Tensor) -> Tensor:
    sq = g.diagonal()
    return (sq.unsqueeze(0) + sq.unsqueeze(1) - 2.0 * g).clamp_min(0.0)


def row_norms(stacked: Tensor) -> Tensor:
    if _use_native(stacked):
        return _EXT.row_norms(stacked.view(1, -1) if stacked.dim() == 1 else stacked).view(
            () if stacked.dim() == 1 else (-1,)
        )
    return ref.row_norms(stacked)


def l2_dists_to(own: Tensor, stacked: Tensor) -> Tensor:
    if _use_native(stacked):
        return _EXT.l2_dists_to(own, stacked)
    return ref.l2_dists_to(own, stacked)


# ------------------------------------------------------------------ K3
def krum_scores(d2: Tensor, num_compromised: int) -> Tensor:
    # m x m is tiny (m <= nodes); torch path is fine on both devices.
    return ref.krum_scores(d2, num_compromised)


def krum_select(d2: Tensor, num_compromised: int) -> Tensor:
    return ref.krum_select(d2, num_compromised)


# ------------------------------------------------------------------ K4/K5
def _packed_sketch_table(hash_idx: Tensor, signs: Tensor, device) -> Tensor:
    """hash+sign packed into one int32 per element (bin in the low 31 bits,
    sign in the sign bit) — halves the kernel's table traffic. Cached on the
    hash tensor (the aggregator reuses its seeded tables every round)."""
    packed = getattr(hash_idx, "_murmura_packed", None)
    if packed is None or packed.device != device:
        neg = (signs < 0).to(torch.int32)
        packed = (hash_idx.to(torch.int32) | (neg << 31)).to(device).contiguous()
        try:
            hash_idx._murmura_packed = packed
        except Exception:
            pass
    return packed


def _grouped_sketch_tables(hash_idx: Tensor, signs: Tensor, device):
    """Detect group-of-8-constant bins (ops.make_sketch_tables' layout) and
    build the packed group table: bin | signbits<<16 per group, plus a
    per-element packed tail for P % 8 leftovers. Cached on the hash tensor."""
    cached = getattr(hash_idx, "_murmura_g8", None)
    if cached is not None and cached[0].device == device:
        return cached
    P = hash_idx.numel()
    ng = P // 8
    if ng == 0 or int(hash_idx.max()) >= (1 << 16):
        return None
    h8 = hash_idx[: ng * 8].view(ng, 8)
    if not bool((h8 == h8[:, :1]).all()):
        return None
    neg = (signs[: ng * 8].view(ng, 8) < 0).to(torch.int32)
    bits = (neg << (16 + torch.arange(8, dtype=torch.int32, device=neg.device))).sum(
        dim=1, dtype=torch.int32
    )
    gt = (h8[:, 0].to(torch.int32) | bits).to(device).contiguous()
    tneg = (signs[ng * 8 :] < 0).to(torch.int32)
    tail = (hash_idx[ng * 8 :].to(torch.int32) | (tneg << 31)).to(device).contiguous()
    out = (gt, tail)
    try:
        hash_idx._murmura_g8 = out
    except Exception:
        pass
    return out


def count_sketch(stacked: Tensor, hash_idx: Tensor, signs: Tensor, sketch_size: int) -> Tensor:
    if _use_native(stacked if stacked.dim() == 2 else stacked.view(1, -1)):
        x = stacked if stacked.dim() == 2 else stacked.view(1, -1)
        if x.shape[0] * sketch_size * 4 <= 64 * 1024 and sketch_size < (1 << 16):
            g8 = _grouped_sketch_tables(hash_idx, signs, x.device)
            if g8 is not None:
                out = _EXT.count_sketch_g8(x, g8[0], g8[1], sketch_size)
                return out if stacked.dim() == 2 else out.view(-1)
        pt = _packed_sketch_table(hash_idx, signs, x.device)
        out = _EXT.count_sketch(x, pt, sketch_size)
        return out if stacked.dim() == 2 else out.view(-1)
    return ref.count_sketch(stacked, hash_idx, signs, sketch_size)


make_sketch_tables = ref.make_sketch_tables


# ------------------------------------------------------------------ K6
def sgd_step(flat_params: Tensor, grad: Tensor, lr: float) -> None:
    if _use_native(flat_params):
        _EXT.sgd_step(flat_params, grad, lr)
        return
    ref.sgd_step(flat_params, grad, lr)


def sgd_step_lrt(flat_params: Tensor, grad: Tensor, lr: Tensor) -> None:
    """K6 with a device-tensor lr (hipGraph-capturable)."""
    if _use_native(flat_params):
        _EXT.sgd_step_lrt(flat_params, grad, lr)
        return
    flat_params.add_(grad * (-lr))


# ------------------------------------------------------------------ K7
def ce_loss_acc(logits: Tensor, targets: Tensor) -> Tuple[Tensor, Tensor]:
    if _use_native(logits):
        out = _EXT.ce_loss_acc(logits, targets)
        return out[0], out[1]
    return ref.ce_loss_acc(logits, targets)


# ------------------------------------------------------------------ K8
def evidential_stats(logits: Tensor, targets: Tensor):
    if _use_native(logits):
        out = _EXT.evidential_stats(logits, targets)
        return out[0], out[1], out[2], out[3]
    return ref.evidential_stats(logits, targets)


# ------------------------------------------------------------------ K10
def gaussian_inject(flat: Tensor, noise_std: float, seed: int, offset: int = 0) -> Tensor:
    if _use_native(flat):
        return _EXT.gaussian_inject(flat, noise_std, seed, offset)
    return ref.gaussian_inject(flat, noise_std, seed, offset)


# ------------------------------------------------------------------ K11
def scale_inject(flat: Tensor, lam: float) -> Tensor:
    if _use_native(flat):
        return _EXT.scale_inject(flat, lam)
    return ref.scale_inject(flat, lam)


# ------------------------------------------------- under torch.vmap (K16, K18)
_transforms_active = torch._C._are_functorch_transforms_active


def _is_mapped(*tensors: Optional[Tensor]) -> bool:
    """Whether torch.vmap, where a transform is active, is at work on one of them: those have no
    memory that a kernel could read."""
    functorch = torch._C._functorch
    return functorch.peek_interpreter_stack().key() == functorch.TransformType.Vmap and any(
        t is not None and functorch.is_batchedtensor(t) for t in tensors)


def _one_by_one(op, info, in_dims, args):
    """The mapped call as one call for each element, so that each has the results that it has alone."""
    return torch.stack([
        op(*(a if d is None else a.select(d, i) for a, d in zip(args, in_dims)))
        for i in range(info.batch_size)
    ]), 0


class _MappedGroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(x, num_groups, weight, bias, eps, act, res):
        return group_norm_act(x, num_groups, weight, bias, eps, act, res)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def vmap(info, in_dims, *args):
        return _one_by_one(group_norm_act, info, in_dims, args)


class _MappedLinearAct(torch.autograd.Function):
    @staticmethod
    def forward(x, weight, bias, act, res):
        return linear_act(x, weight, bias, act, res)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def vmap(info, in_dims, *args):
        return _one_by_one(linear_act, info, in_dims, args)


# ------------------------------------------------------------------ K16
def group_norm_act(x: Tensor, num_groups: int, weight: Optional[Tensor] = None,
                   bias: Optional[Tensor] = None, eps: float = 1e-5, act: str = "none",
                   res: Optional[Tensor] = None) -> Tensor:
    """Group norm, residual and activation in one: y = act(norm(x) * weight +
    bias + res), differentiable in x, weight, bias and res.

    x is [N, C, H, W] or [N, C], fp32 or bf16; images are worked on channels
    last (another layout is copied first) and y comes back so. weight and bias
    ([C]) are of x's type or fp32, res is like x. act: "none", "relu", "silu"
    or "gelu" (by erf). Statistics are held in fp32 and belong to each sample
    alone: nothing is kept between calls. Under torch.vmap each element is a
    call; other transforms, and a derivative going forward, are refused on a GPU."""
    ref.check_group_norm_act(x, num_groups, weight, bias, res)
    code = ref.check_act(act)
    if _transforms_active() and _is_mapped(x, weight, bias, res):
        return _MappedGroupNormAct.apply(x, num_groups, weight, bias, eps, act, res)
    if _use_native(x):
        return _EXT.group_norm_act(x, num_groups, weight, bias, eps, code, res)
    return ref.group_norm_act(x, num_groups, weight, bias, eps, act, res)


# ------------------------------------------------------------------ K17
def adamw_state(numel: int, device, bits: int = 32):
    """(exp_avg, exp_avg_sq, step) of an optimizer that has done no step: the
    moments of ``numel`` parameters in 32 bits, or in 8 with an exponent for
    each 256 values, and the count of steps on the device."""
    if bits not in (8, 32):
        raise ValueError(f"adamw_state: moments are held in 8 or 32 bits, not {bits}")

    def moment():
        if bits == 32:
            return torch.zeros(numel, dtype=torch.float32, device=device)
        return (torch.zeros(numel, dtype=torch.uint8, device=device),
                torch.zeros(-(-numel // ref.ADAMW_BLOCK), dtype=torch.uint8, device=device))

    return moment(), moment(), torch.zeros(1, dtype=torch.int64, device=device)


def adamw_step(params: Union[Tensor, Sequence[Tensor]], grads: Union[Tensor, Sequence[Tensor]],
               exp_avg: ref.Moment, exp_avg_sq: ref.Moment, step: Tensor,
               lr: Union[float, Tensor], betas: Tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.01, seed: int = 0) -> None:
    """One AdamW step over all tensors of a model, in place.

    params: a flat vector or the tensors of a model, fp32 or bf16, without gaps
    or shared memory; grads: as many, of the same shapes, of their type or
    fp32 (a gradient with other strides than its parameter's is copied first).
    exp_avg, exp_avg_sq, step: as ``adamw_state`` makes them, the moments in the
    order of the parameters' memory. lr: a number, or one fp32 value on the device,
    which a captured step reads anew on each replay; the step's count too lives on
    the device. bf16 parameters and 8-bit moments are rounded up with the
    probability of what is cut off, by a hash of (seed, step, place): runs repeat
    bit for bit, and ranks or nodes that shall differ take different seeds.

    A refused call leaves everything as it was. On a GPU, 8-bit moments refuse
    over 160 tensors within 256 values: such small ones are passed as one."""
    params, grads = ref.as_list(params), ref.as_list(grads)
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"adamw_step: betas lie in [0, 1), got {betas}")
    if params and _use_native(params[0]):
        on_device = isinstance(lr, Tensor)
        _EXT.adamw_step(
            params, grads, [exp_avg] if isinstance(exp_avg, Tensor) else list(exp_avg),
            [exp_avg_sq] if isinstance(exp_avg_sq, Tensor) else list(exp_avg_sq), step,
            0.0 if on_device else lr, lr if on_device else None, betas[0], betas[1], eps,
            weight_decay, seed & 0xFFFFFFFF)
        return
    ref.adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr, betas, eps, weight_decay, seed)


def adamw_dequantize(exp_avg: ref.Moment, exp_avg_sq: ref.Moment,
                     dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor]:
    """The values of 8-bit moments, in fp32 or bf16 (which holds them as they are)."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"adamw_dequantize: fp32 or bf16, not {dtype}")
    if isinstance(exp_avg, Tensor) or isinstance(exp_avg_sq, Tensor):
        raise ValueError("adamw_dequantize: moments of 8 bits are (codes, exponents); those of 32 "
                         "are values already")
    if _use_native(exp_avg[0]):
        return _EXT.adamw_decode(list(exp_avg), list(exp_avg_sq), dtype == torch.bfloat16)
    return (ref.adamw_decode(*exp_avg, True).to(dtype), ref.adamw_decode(*exp_avg_sq, False).to(dtype))


# ------------------------------------------------------------------ K18
def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: str = "none",
               res: Optional[Tensor] = None) -> Tensor:
    """Matrix product with its epilogue: y = act(x @ weight.T + bias + res),
    differentiable in all four.

    x is [..., K], weight [N, K] (``nn.Linear``'s layout), fp32 or bf16, of one
    type; bias [N] of that type or fp32; res like y. act: "none", "relu",
    "silu" or "gelu" (by erf). Sums are fp32, also over bf16 products. For the
    backward pass silu and gelu keep what they are taken of, in x's type. Under
    torch.vmap, on a GPU, each element is a call; other transforms, and a
    derivative going forward, are refused there."""
    ref.check_linear_act(x, weight, bias, res)
    code = ref.check_act(act)
    if _use_native(x):
        if _transforms_active() and _is_mapped(x, weight, bias, res):
            return _MappedLinearAct.apply(x, weight, bias, act, res)
        return _EXT.linear_act(x, weight, bias, code, res)
    return ref.linear_act(x, weight, bias, act, res)
