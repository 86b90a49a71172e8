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


def test_sums_over_many_parts_are_no_long_chains(gpu):
    """A parameter's gradient is joined from 65 536 stretches of 128 tokens here. Positive values that are all alike round the same way
    every time; a path to the result has at most 128 additions of tokens and two levels of 64 + 16 of stretches, each of which
    rounds by half a unit in the last place, 2^-24, of a partial sum that is no larger than the whole."""
    batch, T, value = 64, 131072, 1.990972876548767
    x = torch.ones(batch, T, 8, device=gpu)
    w, b = torch.randn(8, 4, device=gpu, requires_grad=True), torch.randn(8, device=gpu, requires_grad=True)
    gw, gb = torch.autograd.grad(f.causal_conv(x, w, b), (w, b), torch.full_like(x, value))
    value = float(torch.tensor(value))  # (as float32 holds it)
    bound = (128 + 2 * (64 + 16)) * 2.0 ** -24
    for k in range(4):  # (tap k reads no token for the first 3 - k)
        want = value * batch * (T - (3 - k))
        assert (gw[:, k].double() - want).abs().max() <= bound * want, k
    want = value * batch * T
    assert (gb.double() - want).abs().max() <= bound * want
