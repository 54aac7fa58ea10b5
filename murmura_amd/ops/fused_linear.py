"""Linear layer with bias, residual and activation in the product's epilogue
(K18), as a module with ``nn.Linear``'s parameters and state-dict names."""

from __future__ import annotations

from typing import Optional

from torch import Tensor, nn

from murmura_amd import ops


class MurmuraLinear(nn.Linear):
    """y = act(x W^T + b (+ res))."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 act: str = "none"):
        super().__init__(in_features, out_features, bias=bias)
        ops.ref.check_act(act)
        self.act = act

    def forward(self, x: Tensor, res: Optional[Tensor] = None) -> Tensor:
        return ops.linear_act(x, self.weight, self.bias, self.act, res)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, act={self.act}"
