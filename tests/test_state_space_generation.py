"""Generation with the state space example (examples/state_space_lm.py) from prompts at the edges."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import state_space_lm as lm  # noqa: E402


def test_as_many_tokens_as_asked_for_after_prompts_that_have_any():
    torch.manual_seed(0)
    model = lm.Model(channels=32, layers=1)
    three = lm.generate(model, [[1, 2, 3], [7]], 3)
    for count in range(3):
        assert lm.generate(model, [[1, 2, 3], [7]], count) == [t[:count] for t in three]
    assert lm.generate(model, [], 2) == []
    for prompts in ([[1, 2, 3], []], [[]]):  # (there is no token whose logits could say what comes first)
        with pytest.raises(ValueError, match="empty"):
            lm.generate(model, prompts, 2)
