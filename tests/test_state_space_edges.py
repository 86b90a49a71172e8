"""
The state space layer's operators at the edges of their arguments, without a GPU.
"""
import torch

from scanscam_amd import baseline, rms_norm


def test_softplus_has_its_gradient_at_zero():
    """The step size's gradient is sigmoid(dt + dt_bias) times what comes in, 1/2 at zero, where projections that start from zeros are."""
    dt = torch.tensor([[[0.0], [-0.0], [1e-30], [3.0], [-90.0], [90.0], [float("-inf")]]], dtype=torch.float64, requires_grad=True)
    x, one, A = torch.ones_like(dt), torch.ones_like(dt), torch.zeros(1, 1, dtype=torch.float64)
    for T in range(dt.shape[1]):
        # With A = 0, B = C = x = 1 the last token adds its own step size to the output, the earlier ones theirs.
        y = baseline.naive_selective_scan(x, dt, A, one, one, softplus=True)
        (g,) = torch.autograd.grad(y[0, T, 0], dt)
        want = torch.sigmoid(dt.detach()) * (torch.arange(dt.shape[1]) <= T)[None, :, None]
        torch.testing.assert_close(g, want, rtol=1e-14, atol=0.0)


def test_eight_bits_of_no_channels():
    """A row without values is a row of zeros: its scale is 1."""
    x = torch.zeros(2, 3, 0)
    q, scale, total = rms_norm(x, torch.zeros(0), x, quant=torch.int8)
    assert q.shape == x.shape and total.shape == x.shape and torch.equal(scale, torch.ones(2, 3))
