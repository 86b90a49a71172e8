"""
The linear attention layer's operators: numbers among their arguments. The same on both devices.
"""
import pytest
import torch

import scanscam_amd as f


def check(device):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g).to(device)  # noqa: E731
    q, v, x = r(1, 4, 2, 8), r(1, 4, 2, 8), r(3, 12)
    want, normed = f.linear_attention(q, q, v, scale=0.5), f.group_norm(x, 3, eps=0.25)
    learned = torch.tensor(0.5, requires_grad=True)
    for other in (torch.tensor(0.5), learned.detach(), torch.tensor(0.5, device=device)):
        assert torch.equal(f.linear_attention(q, q, v, scale=other), want)
        assert torch.equal(f.group_norm(x, torch.tensor(3), eps=other / 2), normed)
    with torch.no_grad():
        assert torch.equal(f.linear_attention(q, q, v, scale=learned), want)
    # A gradient that nobody would get.
    with pytest.raises(TypeError, match="scale"):
        f.linear_attention(q, q, v, scale=learned)
    with pytest.raises(TypeError, match="eps"):
        f.group_norm(x, 3, eps=learned)
    # Not so many groups as a part of a number says.
    for groups in (2.5, 3.0, "3", None):
        with pytest.raises(TypeError):
            f.group_norm(x, groups)


def test_numbers():
    check("cpu")


@pytest.mark.gpu
def test_numbers_on_the_gpu(gpu):
    check(gpu)
