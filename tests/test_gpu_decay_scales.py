"""``decay_linear_attention`` with scales of 0, far below and far above 1, against the recurrence in 64 bits.

With u = 2^-8 (half a step of bf16) and M the result of the inputs' magnitudes: bf16 results within 2.1 u M + u |y|
(each term rounded at most twice on its way, the result once), fp32 ones within 2^-16 M (fewer than 2^8 roundings of
2^-24). What lies below the smallest normal number of fp32, 2^-126, may be flushed: 2^-120 for sums of 2^6 of them."""
import pytest
import torch

from oracle import token as OT
from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8


def _grads(fn, x, douts, cast):
    leaves = [cast(t).clone().requires_grad_(True) for t in x]
    out, final = fn(*leaves)
    return (out.detach(), final.detach(), *torch.autograd.grad((out, final), leaves, [g.to(o.dtype) for g, o in zip(douts, (out, final))]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-42, 1e-30, -1e-12, 1e15])
def test_outputs_and_gradients(dtype, d, scale):
    g = torch.Generator().manual_seed(d)
    n, h = 300, 2
    q, k, v, dout = (torch.randn(1, n, h, d, generator=g).to(DEV, dtype) for _ in range(4))
    log_decay = torch.tensor([-0.02, -0.3], device=DEV)
    initial, dfinal = (torch.randn(1, h, d, d, generator=g).to(DEV) for _ in range(2))
    x, douts = (q, k, v, log_decay, initial), (dout, dfinal)
    own = lambda q, k, v, g, s: W.decay_linear_attention(q, k, v, g, initial_state=s, scale=scale)  # noqa: E731
    plain = lambda f: lambda q, k, v, g, s: OT.decay_linear_attention(q, k, v, g, initial_state=s, scale=f)  # noqa: E731
    got = _grads(own, x, douts, lambda t: t)
    want = _grads(plain(scale), x, douts, torch.Tensor.double)
    size = _grads(plain(abs(scale)), (q.abs(), k.abs(), v.abs(), log_decay, initial.abs()), [t.abs() for t in douts], torch.Tensor.double)
    for name, a, w, m in zip(("out", "final", "dq", "dk", "dv", "dlog_decay", "dinitial"), got, want, size):
        assert torch.isfinite(a).all(), name
        bound = (2.1 * U * m + U * w.abs() if a.dtype == torch.bfloat16 else 2.0 ** -16 * m) + 2.0 ** -120
        assert ((a.double() - w).abs() <= bound).all(), f"{name}: {((a.double() - w).abs() / bound).max().item():.2f} of the bound"
    if scale == 0:
        assert not got[0].any() and not got[2].any()
