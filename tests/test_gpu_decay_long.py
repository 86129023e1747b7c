"""``decay_linear_attention`` where sequences have many segments and segments many tokens, all results and gradients
against the sums over pairs of tokens in 64 bits.

Tolerances. u = 2^-8 is half a step of bf16, M the result that the inputs' magnitudes would have. In bf16 rows a term is
rounded once on its way (its decayed score, or its weighted key where it comes through the running state, which is read
in two parts, 2^-17): 1.05 u M, and u |y| for the result's own rounding. fp32 results come from operands cut in three exact
parts, or from fp32 products: a path of fewer than 300 rounded sums within a segment (1,536 tokens, 16 a product, three
parts: 2^-15.7), the weights' 2^-18 and the carry from segment to segment: 2^-15 M. Roundings are independent, so a whole
tensor's error stays below 1.25 u of its norm in bf16."""
import pytest
import torch

from worldattention_amd import _lib
from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8
NAMES = ("out", "final", "dq", "dk", "dv", "dlog_decay", "dinitial")


def _pairs(q, k, v, log_decay, initial, scale):
    """One sequence, ``[h, n, d]`` in fp64: every token against every one before it."""
    n = q.shape[1]
    t = torch.arange(n, dtype=torch.float64, device=DEV)
    lag = t[:, None] - t
    g = log_decay.view(-1, 1, 1)
    weight = torch.where(lag >= 0, (g * lag.clamp(min=0)).exp(), 0.0)
    start, end = (g * (t + 1)[:, None]).exp(), (g * (n - 1 - t)[:, None]).exp()
    out = scale * ((q @ k.transpose(1, 2).contiguous() * weight) @ v + start * (q @ initial))
    return out, (k * end).transpose(1, 2).contiguous() @ v + (g * n).exp() * initial


def _reference(x, douts, lengths, cast):
    """Results and gradients, 8 heads of a sequence at a time."""
    q, k, v, log_decay, initial = (cast(t.detach().double()) if i != 3 else t.detach().double() for i, t in enumerate(x))
    dout, dfinal = (cast(t.double()) for t in douts)
    want = [torch.zeros_like(t) for t in (v, initial, q, k, v, log_decay, initial)]
    for b, n in enumerate(lengths):
        for h0 in range(0, q.shape[2], 8):
            hs = slice(h0, h0 + 8)
            part = [t[b, :n, hs].transpose(0, 1).contiguous().requires_grad_(True) for t in (q, k, v)]
            part += [log_decay[hs].clone().requires_grad_(True), initial[b, hs].clone().requires_grad_(True)]
            out, final = _pairs(*part, q.shape[-1] ** -0.5)
            grads = torch.autograd.grad((out, final), part, (dout[b, :n, hs].transpose(0, 1), dfinal[b, hs]))
            want[0][b, :n, hs], want[1][b, hs] = out.detach().transpose(0, 1), final.detach()
            for w, d in zip(want[2:5], grads[:3]):
                w[b, :n, hs] = d.transpose(0, 1)
            want[5][hs] += grads[3]
            want[6][b, hs] = grads[4]
    return want


# segments x tokens of one, with and without derivatives: many short ones (the carry's and the launch's dealing pass
# eight), few long ones (several 256-token units and groups, several spans), an odd tail in each
@pytest.mark.parametrize("b,n,h,d,dtype,lengths,segments,derivs", [
    (1, 2101, 2, 128, torch.bfloat16, None, 17, 17), (2, 1301, 1, 64, torch.bfloat16, (1301, 1077), 11, 11),
    (1, 1349, 3, 64, torch.float32, None, 11, 11), (2, 1190, 1, 128, torch.float32, (1190, 1025), 10, 10),
    (4, 2101, 32, 128, torch.bfloat16, (2101, 1500, 1088, 333), 2, 2), (2, 1099, 128, 64, torch.bfloat16, (1099, 515), 1, 1),
    (1, 3001, 128, 128, torch.bfloat16, None, 2, 4), (2, 1099, 64, 128, torch.float32, (1099, 700), 2, 2)])
def test_results_and_gradients(b, n, h, d, dtype, lengths, segments, derivs):
    assert [_lib.lib().wa_decay_segments(b, n, h, x) for x in (0, 1)] == [segments, derivs]
    g = torch.Generator().manual_seed(n)
    q, k, v, dout = (torch.randn(b, n, h, d, generator=g).to(DEV, dtype) for _ in range(4))
    log_decay = -torch.exp2(-3 - 8 * torch.rand(h, generator=g)).to(DEV)      # memories of 8 to 2,048 tokens
    log_decay[0] = 0
    initial, dfinal = (torch.randn(b, h, d, d, generator=g).to(DEV) for _ in range(2))
    x, douts, given = (q, k, v, log_decay, initial), (dout, dfinal), lengths
    if lengths is not None:
        given = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    lengths = lengths or (n,) * b
    leaves = [t.clone().requires_grad_(True) for t in x]
    out, final = W.decay_linear_attention(*leaves[:4], initial_state=leaves[4], lengths=given)
    got = (out.detach(), final.detach(), *torch.autograd.grad((out, final), leaves, douts))
    want, size = (_reference(x, douts, lengths, cast) for cast in (lambda t: t, torch.abs))
    for name, a, w, m in zip(NAMES, got, want, size):
        rounded = a.dtype == torch.bfloat16
        bound = (1.05 * U * m + U * w.abs() if rounded else 2.0 ** -15 * m) + 1e-30
        over = ((a.double() - w).abs() / bound).max().item()
        assert over <= 1, f"{name}: {over:.2f} of the bound"
        if rounded:
            assert (a.double() - w).norm() <= 1.25 * U * w.norm(), name
    with torch.no_grad():      # the plan without derivatives
        plain = W.decay_linear_attention(q, k, v, log_decay, initial_state=initial, lengths=given)
    for a, w, m in zip(plain, want, size):
        bound = (1.05 * U * m + U * w.abs() if a.dtype == torch.bfloat16 else 2.0 ** -15 * m) + 1e-30
        assert ((a.double() - w).abs() <= bound).all()
    # fixed decays: gradients of the plan without derivatives
    leaves = [t.clone().requires_grad_(i != 3) for i, t in enumerate(x)]
    out, final = W.decay_linear_attention(*leaves[:4], initial_state=leaves[4], lengths=given)
    fixed = torch.autograd.grad((out, final), [t for t in leaves if t.requires_grad], douts)
    for name, a, w, m in zip(NAMES[2:5] + NAMES[6:], fixed, want[2:5] + want[6:], size[2:5] + size[6:]):
        bound = (1.05 * U * m + U * w.abs() if a.dtype == torch.bfloat16 else 2.0 ** -15 * m) + 1e-30
        assert ((a.double() - w).abs() <= bound).all(), name
