"""
The state space layer's operators at sizes that few calls have: none of something, very many of something, tensors far apart.
"""
import pytest
import torch

import scanscam_amd as f

pytestmark = pytest.mark.gpu


def spoil(gpu, numbers):
    """Leaves memory that the next allocations get in a state that is not zeros."""
    for n in numbers:
        torch.full((n,), float("nan"), device=gpu)


def test_selections_of_no_channels_have_gradients_of_zero(gpu):
    B, C = (torch.randn(2, 5, 4, device=gpu, requires_grad=True) for _ in range(2))
    y = f.selective_scan(torch.empty(2, 5, 0, device=gpu), torch.empty(2, 5, 0, device=gpu), torch.empty(0, 4, device=gpu), B, C)
    spoil(gpu, [B.numel()] * 8)
    for g in torch.autograd.grad(y.sum(), (B, C)):
        assert torch.equal(g, torch.zeros_like(B))
