"""The state space operators as a model uses them together (examples/state_space_lm.py): it learns, and a prompt taken in at once, packed
with others, leaves the states that its tokens one by one leave."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import state_space_lm as lm  # noqa: E402

DEVICES = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="gpu", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_prompts_and_single_tokens_agree(device):
    torch.manual_seed(1)
    model = lm.Model(channels=32, layers=2).to(device)
    prompts = [[3, 1, 2], list(range(1, 20)), [7]]
    with torch.no_grad():
        offsets = torch.tensor([0, 3, 22, 23], dtype=torch.int32, device=device)
        packed = torch.tensor([t for p in prompts for t in p], device=device).unsqueeze(0)
        logits, states = model(packed, offsets=offsets, keep=True)
        for s, (p, end) in enumerate(zip(prompts, (3, 22, 23))):
            like = torch.zeros(1, device=device)
            mine = [layer.new_states(1, like) for layer in model.layers]
            for t in p:
                last = model.step(torch.tensor([t], device=device), mine)
            torch.testing.assert_close(last[0], logits[0, end - 1], rtol=1e-4, atol=1e-4)
            for (kept, state), (kept_packed, state_packed) in zip(mine, states):
                torch.testing.assert_close(kept[0], kept_packed[s], rtol=1e-4, atol=1e-4)
                torch.testing.assert_close(state[0], state_packed[s], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("device", DEVICES)
def test_a_step_of_training_has_every_gradient(device):
    torch.manual_seed(2)
    model = lm.Model(channels=32, layers=1).to(device)
    losses = lm.train(model, 3, device, batch=2, T=12)
    assert losses[-1] < losses[0]
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0 for p in model.parameters())


@pytest.mark.gpu
def test_the_example_learns(gpu, capsys):
    losses, out = lm.main(["--device", "cuda", "--steps", "120", "--dtype", "bfloat16"])
    assert losses[-1] < 0.5 * losses[0]
    assert "3 of 3" in capsys.readouterr().out and len(out) == 3
