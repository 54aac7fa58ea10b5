"""Calls of the local training step's operators beside the ordinary ones."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from murmura_amd import ops

FP32 = torch.float32


def _randn(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("lead", [(), (6,), (2, 3), (2, 1, 4)])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_inputs_changed_in_place_are_noticed(lead, act):
    base, w = _randn((*lead, 8), FP32, 1).cuda(), _randn((5, 8), FP32, 2).cuda().requires_grad_(True)
    # what the weight's gradient reads
    x = base.clone()
    y = ops.linear_act(x, w, act=act)
    x.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), w)
    # what the input's gradient reads
    x, v = base.clone().requires_grad_(True), w.detach().clone()
    y = ops.linear_act(x, v, act=act)
    v.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), x)
    # a copy that the call made of columns is its own
    x = base.new_zeros(*lead, 16)[..., ::2]
    x.copy_(base)
    want, = torch.autograd.grad(ops.linear_act(base, w, act=act).sum(), w)
    y = ops.linear_act(x, w, act=act)
    got, = torch.autograd.grad(y.sum(), w)
    assert torch.equal(got, want)
