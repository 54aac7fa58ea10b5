"""A node's AdamW state over its flat-bound parameters (K17).

The reference trains with plain SGD only (reference: murmura/core/node.py:74);
SGD stays the default. With ``training.optimizer: adamw`` a node keeps its two
moments and its count of steps beside its parameters, on the same device, in
fp32 or in 8 bits (8 or 2 bytes a parameter: many simulated nodes share one
GPU). Aggregation replaces parameters and leaves the moments as they are: they
describe the node's own data.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Sequence, Tuple

import torch
from torch import Tensor

from murmura_amd import ops


@dataclass(frozen=True)
class AdamWConfig:
    betas: Tuple[float, float] = (0.9, 0.999)
    eps: float = 1e-8
    weight_decay: float = 0.01
    state_bits: int = 32  # 32 or 8
    seed: int = 0  # of the rounding of bf16 parameters and 8-bit moments


class NodeAdamW:
    """Moments and steps of the trainable parameters ``params`` (views of a
    FlatParamStore, so the tensors here stay valid for the node's life)."""

    def __init__(self, params: Sequence[Tensor], config: AdamWConfig):
        self.params = [p.detach() for p in params]
        self.config = config
        numel = sum(p.numel() for p in self.params)
        self.exp_avg, self.exp_avg_sq, self.count = ops.adamw_state(
            numel, self.params[0].device, config.state_bits
        )

    @torch.no_grad()
    def step(self, grads: Sequence[Tensor], lr: float) -> None:
        c = self.config
        ops.adamw_step(self.params, grads, self.exp_avg, self.exp_avg_sq, self.count, lr,
                       betas=c.betas, eps=c.eps, weight_decay=c.weight_decay, seed=c.seed)

    def tensors(self) -> List[Tensor]:
        """All state, in a fixed order."""
        out: List[Tensor] = []
        for moment in (self.exp_avg, self.exp_avg_sq):
            out += [moment] if isinstance(moment, Tensor) else list(moment)
        return out + [self.count]

    def state_payload(self) -> Dict[str, object]:
        return {"bits": self.config.state_bits,
                "tensors": [t.detach().cpu().clone() for t in self.tensors()]}

    def load_payload(self, payload: Dict[str, object]) -> None:
        mine, saved = self.tensors(), payload["tensors"]
        if payload["bits"] != self.config.state_bits or [t.shape for t in mine] != [
                t.shape for t in saved]:
            raise ValueError(
                f"optimizer state of {payload['bits']} bits and {saved[0].numel()} parameters "
                f"does not fit {self.config.state_bits} bits and {mine[0].numel()}")
        for t, s in zip(mine, saved):
            t.copy_(s)
