"""What autograd sees of the token-by-token operators' in-place calls."""
import pytest
import torch

from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_step_counts_as_a_change_of_its_state():
    """A graph that saved the state must not go backwards through what a step has made of it."""
    state = torch.randn(2, 3, 64, 64, device=DEV)
    w = torch.randn_like(state).requires_grad_(True)
    x = [torch.randn(2, 1, 3, 64, device=DEV) for _ in range(3)]
    loss = (w * state).sum()
    before = state._version
    with torch.no_grad():
        W.decay_linear_step(*x, torch.full((3,), -0.1, device=DEV), state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_steps_under_inference_mode():
    with torch.inference_mode():
        state = torch.randn(1, 2, 64, 64, device=DEV)
        kept = state.clone()
        x = [torch.randn(1, 1, 2, 64, device=DEV) for _ in range(3)]
        out = W.decay_linear_step(*x, torch.full((2,), -0.1, device=DEV), state)
    assert out.shape == (1, 1, 2, 64) and not torch.equal(state, kept)
