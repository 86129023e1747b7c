"""What autograd sees of the token-by-token operators' in-place and empty calls."""
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,n,h,d,dv", [(2, 0, 3, 64, 64), (0, 5, 3, 64, 64), (2, 5, 0, 64, 64), (2, 0, 3, 48, 80), (2, 0, 3, 16, 5),
                                       (2, 5, 3, 0, 16), (2, 5, 3, 16, 0)])
@pytest.mark.parametrize("asked", ["q", "k", "v", "log_decay", "initial", "all"])
def test_gradients_of_empty_calls(dtype, b, n, h, d, dv, asked):
    """No tokens, sequences, heads or channels: the state passes through (its gradient too), the other gradients are 0."""
    x = {"q": torch.randn(b, n, h, d, device=DEV).to(dtype), "k": torch.randn(b, n, h, d, device=DEV).to(dtype),
         "v": torch.randn(b, n, h, dv, device=DEV).to(dtype), "log_decay": -torch.rand(h, device=DEV),
         "initial": torch.randn(b, h, dv, d, device=DEV).transpose(2, 3)}
    leaves = {m: t.detach().requires_grad_(asked in (m, "all")) for m, t in x.items()}
    out, final = W.decay_linear_attention(leaves["q"], leaves["k"], leaves["v"], leaves["log_decay"], initial_state=leaves["initial"])
    assert out.shape == (b, n, h, dv) and out.dtype == dtype and torch.equal(final, x["initial"]) and final.is_contiguous()
    want = [t for t in leaves.values() if t.requires_grad]
    dfinal = torch.randn_like(final)
    got = torch.autograd.grad((out, final), want, (torch.zeros_like(out), dfinal))
    for leaf, g in zip(want, got):
        assert g.shape == leaf.shape and g.dtype == leaf.dtype
        assert torch.equal(g, dfinal) if leaf is leaves["initial"] else not g.any()
    # the state of such a prompt goes on into a step
    if n == 0 and b:
        with torch.no_grad():
            W.decay_linear_step(*(torch.randn(b, 1, h, w, device=DEV).to(dtype) for w in (d, d, dv)), x["log_decay"], final.detach())
