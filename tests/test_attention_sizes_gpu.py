"""
The attention layer's operators at sizes that few calls have: none of something, very many of something.
"""
import pytest
import torch

import scanscam_amd as f
from test_state_space_sizes_gpu import spoil

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("state", [False, True])
def test_queries_and_keys_of_no_heads_have_gradients_of_zero(gpu, dtype, state):
    q, k = (torch.randn(2, 5, 3, 4, device=gpu).to(dtype).requires_grad_() for _ in range(2))
    v = torch.empty(2, 5, 0, 6, dtype=dtype, device=gpu)
    s = torch.empty(2, 0, 4, 6, device=gpu) if state else None
    for offsets in (None, torch.tensor([0, 2, 5], device=gpu)):
        n = 2 if offsets is None else 1
        y, new = f.linear_attention(q[:n], k[:n], v[:n], torch.zeros(0, device=gpu), state=s, offsets=offsets, return_state=True)
        assert y.shape == (n, 5, 0, 6) and new.shape == (2, 0, 4, 6)
        spoil(gpu, [q.numel(), q.numel() // 2] * 8)
        for g in torch.autograd.grad(y.sum() + new.sum(), (q, k)):
            assert torch.equal(g, torch.zeros_like(q))


def test_very_many_sequences(gpu):
    """More heads of sequences than a launch has workgroups, single tokens of more rows."""
    n = (1 << 22) + 3
    g = torch.Generator(device=gpu).manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=gpu)  # noqa: E731
    q, k, v, decay, state = r(n, 1, 1, 2), r(n, 1, 1, 2), r(n, 1, 1, 3), -r(n, 1, 1).abs(), r(n, 1, 2, 3)
    leaves = [t.requires_grad_() for t in (q, k, v, decay, state)]
    y, new = f.linear_attention(q, k, v, decay, state=state, return_state=True)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    s = wide[3].exp()[..., None] * wide[4] + wide[1][:, 0].unsqueeze(-1) * wide[2][:, 0].unsqueeze(-2)
    want = (wide[0][:, 0].unsqueeze(-1) * s).sum(-2).unsqueeze(1)
    gy, gs = r(*y.shape), r(*new.shape)
    # (a token's sums are of two or three products, at some ten roundings each)
    close = lambda a, b: (a.double() - b).abs().max() <= 2.0 ** -19 * b.abs().max()  # noqa: E731
    assert close(y, want) and close(new, s)
    for a, b in zip(torch.autograd.grad((y, new), leaves, (gy, gs)), torch.autograd.grad((want, s), wide, (gy.double(), gs.double()))):
        assert close(a, b)
    n = (1 << 24) + 5
    q, k, v, state = r(n, 1, 1), r(n, 1, 1), r(n, 1, 1), r(n, 1, 1, 1)
    want = (state.double() + (k * v).double().unsqueeze(-1))
    y = f.linear_attention_step(state, q, k, v)
    assert close(state, want) and close(y, q.double() * want[..., 0])
