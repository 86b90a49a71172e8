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


@pytest.mark.parametrize("quant", [torch.int8, torch.float8_e4m3fn])
def test_eight_bits_of_no_channels(gpu, quant):
    """A row without values is a row of zeros: its scale is 1."""
    x, w = torch.empty(5, 60, 0, device=gpu, dtype=torch.bfloat16), torch.empty(0, device=gpu)
    spoil(gpu, [300] * 8)
    q, scale = f.rms_norm(x, w, quant=quant)
    assert q.shape == x.shape and torch.equal(scale, torch.ones(5, 60, device=gpu))
    spoil(gpu, [300] * 8)
    q, scale, total = f.rms_norm(x, w, x.float(), quant=quant)
    assert total.shape == x.shape and torch.equal(scale, torch.ones(5, 60, device=gpu))
