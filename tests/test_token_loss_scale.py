"""Upstream gradients as large as loss scaling makes them."""
import math

import pytest
import torch

from dear_pytorch_amd.ops.token_loss import token_logprobs


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("V", [40, 30528])
def test_entropy_gradient_scales_with_ruled_out_tokens(V, dev):
    """A power of two more: the same digits, also next to tokens of -inf and of
    the type's lowest value, whose own gradient is 0."""
    gen = torch.Generator().manual_seed(V)
    z = torch.randn(3, V, generator=gen)
    z[0, ::2], z[1, ::3] = -math.inf, torch.finfo(torch.float32).min
    z = z.to(dev).requires_grad_(True)

    def grad(scale):
        h = token_logprobs(z, None).entropy
        return torch.autograd.grad(h, z, torch.full_like(h, scale))[0]

    one = grad(1.0)
    assert torch.isfinite(one).all() and (one[0, ::2] == 0).all()
    for power in (10, 16, 30, 60):
        assert torch.equal(grad(2.0 ** power), one * 2.0 ** power), power
