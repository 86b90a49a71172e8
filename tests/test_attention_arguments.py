"""
The linear attention layer's operators: numbers among their arguments, on both devices the same; and states that were made in inference mode.
"""
import pytest
import torch

import scanscam_amd as f
from scanscam_amd import attention, state_space


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


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_states_made_in_inference_mode(gpu, monkeypatch, native):
    """They have no version to count up: steps change them as others, inside of the mode and outside."""
    if not native:
        monkeypatch.setattr(attention, "_native", None)
        monkeypatch.setattr(state_space, "_native", None)
    g = torch.Generator(device=gpu).manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
    q, v, x, A, B, w = r(2, 2, 8), r(2, 2, 8), r(2, 6), -r(6, 4).abs(), r(2, 4), r(6, 3)
    steps = {(2, 2, 8, 8): lambda s: f.linear_attention_step(s, q, q, v), (2, 6, 4): lambda s: f.selective_scan_step(s, x, x, A, B, B), (2, 2, 6): lambda s: f.causal_conv_step(s, x, w)}
    for shape, step in steps.items():
        want = torch.ones(shape, device=gpu)
        ys = [step(want), step(want)]
        with torch.inference_mode():
            state = torch.ones(shape, device=gpu)
            first = step(state).clone()
        with torch.no_grad():
            second = step(state)
        assert torch.equal(state, want) and torch.equal(first, ys[0]) and torch.equal(second, ys[1])
