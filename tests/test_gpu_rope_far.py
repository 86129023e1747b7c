"""``rope_axes`` at positions up to the ends of int64, against exact angles (integers and fractions).

Tolerance: half a step of the output's type and 2^-20 of the pair's largest magnitude for the fp32 part (the reduced angle
rounded to fp32, 2^-26 of a revolution; the sine and cosine, 2 ulp; two products and a sum)."""
import math
from fractions import Fraction

import pytest
import torch

from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")
PLACES = [0, 1, -1, 2**31 - 1, -2**31, 2**40 + 1, -2**40 - 3, 2**53 - 1, 2**53 + 1, -2**60 - 12345, 2**62 + 3, 2**63 - 1, -2**63]


def _turn(position, frequency):
    """The angle in [-pi, pi], from the exact product."""
    rev = Fraction(position) * Fraction(frequency) / TWO_PI
    return float((rev - round(rev)) * TWO_PI)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_any_position(dtype, interleaved):
    sections = (9, 7)
    pairs, n, d = sum(sections), len(PLACES), 40
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, n, 2, d, generator=g).to(dtype)
    pos = torch.tensor([PLACES, PLACES[::-1]]).T.contiguous()
    inv, _ = W.axis_frequencies(2 * pairs, axes=1)
    inv[0], inv[9], inv[3] = 1.0, 0.7071, math.pi / 4
    axis = [0] * sections[0] + [1] * sections[1]
    angle = torch.tensor([[_turn(int(pos[t, axis[p]]), inv[p].item()) for p in range(pairs)] for t in range(n)], dtype=torch.float64)
    c, s = angle.cos()[None, :, None], angle.sin()[None, :, None]
    f = x.double()
    re, im = (f[..., 0:2 * pairs:2], f[..., 1:2 * pairs:2]) if interleaved else (f[..., :pairs], f[..., pairs:2 * pairs])
    turned = (re * c - im * s, re * s + im * c)
    want = torch.cat((torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1), f[..., 2 * pairs:]), -1)
    got = W.rope_axes(x.to(DEV), pos.to(DEV), inv.to(DEV), sections, interleaved=interleaved).cpu()
    bound = torch.finfo(dtype).eps / 2 * 1.01 * want.abs() + 2.0 ** -20 * 2 * f.abs().amax(-1, keepdim=True)
    off = ((got.double() - want).abs() / bound).amax((0, 2, 3))
    assert (off <= 1).all(), dict(zip(PLACES, off.tolist()))
    fits = [i for i, p in enumerate(PLACES) if -2**31 <= p < 2**31]
    narrow = [W.rope_axes(x[:, fits].to(DEV), pos[fits, :1].to(DEV, t), inv[:9].to(DEV), (9,), interleaved=interleaved)
              for t in (torch.int32, torch.int64)]
    assert torch.equal(*narrow)
