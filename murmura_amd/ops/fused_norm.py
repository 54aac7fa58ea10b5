"""Group norm with a fused activation (K16), as a module.

Batch statistics do not travel well between nodes with different data: the
running averages of one node's classes are another's bias. ``MurmuraGroupNorm``
has none. It stands where ``MurmuraBatchNorm2d`` stands (same ``res`` argument,
same fusion of the activation) and keeps ``nn.GroupNorm``'s parameters and
state-dict names.
"""

from __future__ import annotations

from typing import Optional

from torch import Tensor, nn

from murmura_amd import ops


class MurmuraGroupNorm(nn.GroupNorm):
    """y = act(group_norm(x) (+ res)) over [N, C, H, W] (channels last) or [N, C]."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5,
                 affine: bool = True, act: str = "none"):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine)
        ops.ref.check_act(act)
        self.act = act

    def forward(self, x: Tensor, res: Optional[Tensor] = None) -> Tensor:
        return ops.group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps,
                                  self.act, res)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, act={self.act}"
