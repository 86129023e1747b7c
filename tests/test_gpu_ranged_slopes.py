"""Gradients of ``ranged_attention`` whose bias grows with the distance (negative slopes), against 64 bits.

Bounds as those of ``test_gpu_ranged.py``, with u = 2^-8 (half a step of bf16): dS is off by P u E (the output's rounding in delta, E = sum
|o| |do|), by its own rounding u |dS|, and by 2^-11 P (|dP| + |delta|) for the weights (scores of at most 2^8 here); gradients are rounded once more. For
the keys' gradient the weights pass as fp16 with a factor of 2^12: 2^-11 of a weight, or half of fp16's smallest step, 2^-25 2^-12 = 2^-37,
where a weight times the cap's derivative is below 2^-26, as most are where the farthest keys take it all."""
import pytest
import torch

from oracle import ranged as OR
from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8
TINY = 2.0 ** -100


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,h,hk,cap,slopes", [
    (333, 2, 1, None, [-0.3, -0.5]), (1000, 2, 2, None, [-0.1, 0.1]), (1000, 4, 1, 9.0, [-0.1, 0.2, 0.0, -0.2]), (1090, 2, 1, None, [-0.1, -0.09])])
def test_over_a_ragged_last_tile(d, n, h, hk, cap, slopes):
    """The rows behind the last one are no rows: their bias alone passes what an exponential of fp32 holds."""
    g = torch.Generator().manual_seed(n + h)
    q, k, v, do = (torch.randn(1, n, x, d, generator=g).bfloat16().to(DEV) for x in (h, hk, hk, h))
    leaves = [t.requires_grad_(True) for t in (q, k, v, torch.tensor(slopes, device=DEV))]
    out = W.ranged_attention(*leaves[:3], W.key_ranges(1, n, n, device=DEV), cap=cap, slopes=leaves[3])
    grads = torch.autograd.grad(out, leaves, do)
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    y, _, (p, turn, far) = OR.attention(*exact[:3], OR.seen(1, n, n), cap=cap, slopes=exact[3])
    want = torch.autograd.grad((y * do.double()).sum(), exact)
    with torch.no_grad():
        heads = lambda t: t.double().transpose(1, 2).repeat_interleave(h // t.shape[2], 1)  # noqa: E731
        group = lambda t: t.view(1, hk, h // hk, n, d).sum(2).transpose(1, 2)  # noqa: E731
        qh, kh, vh, doh = (heads(t.detach()) for t in (q, k, v, do))
        dp = torch.matmul(doh, vh.transpose(-1, -2).contiguous())
        delta = (p * dp).sum(-1, keepdim=True)
        e = (y.abs() * do.double().abs()).sum(-1).transpose(1, 2)[..., None]
        wide = dp.abs() + delta.abs()
        off = (U + 2.0 ** -10) * p * (dp - delta).abs() + p * U * e + 2.0 ** -11 * p * wide
        small = torch.where(p > 0, 2.0 ** -37 * wide, 0.0)
        bent = (turn + 2.0 ** -20) * d ** -0.5
        bounds = [torch.matmul(off * bent, kh.abs()).transpose(1, 2),
                  group(torch.matmul((off * bent + small * d ** -0.5).transpose(-1, -2).contiguous(), qh.abs())),
                  group(torch.matmul(p.transpose(-1, -2).contiguous(), doh.abs())) * (U + 2.0 ** -11),
                  (2.0 ** -11 * p * wide * far).sum((0, 2, 3))]
    for name, got, w, bound in zip(("dq", "dk", "dv", "dslopes"), grads, want, bounds):
        last = U if name != "dslopes" else 2.0 ** -22
        err = (got.double() - w).abs()
        assert (err <= bound + last * w.abs() + TINY).all(), (name, (err - bound - last * w.abs()).max())
