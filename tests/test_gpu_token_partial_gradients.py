"""Gradients of some of the token-by-token operators' inputs: whatever is asked for, the bits are those of asking for all."""
import itertools

import pytest
import torch

from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decay_gradients_asked_for_one_by_one(dtype):
    g = torch.Generator().manual_seed(6)
    x = [torch.randn(2, 300, 3, 64, generator=g).to(DEV, dtype) for _ in range(3)]
    x += [-torch.rand(3, generator=g).to(DEV), torch.randn(2, 3, 64, 64, generator=g).to(DEV)]
    douts = torch.randn(2, 300, 3, 64, generator=g).to(DEV, dtype), torch.randn(2, 3, 64, 64, generator=g).to(DEV)
    leaves = [t.clone().requires_grad_(True) for t in x]
    results = W.decay_linear_attention(*leaves[:4], initial_state=leaves[4])
    want = torch.autograd.grad(results, leaves, douts, retain_graph=True)
    for some in itertools.chain(itertools.combinations(range(5), 1), itertools.combinations(range(5), 2)):
        got = torch.autograd.grad(results, [leaves[i] for i in some], douts, retain_graph=True)   # of a graph that holds them all
        assert all(torch.equal(a, want[i]) for a, i in zip(got, some)), some
    # frozen inputs: segments are cut another way without the decays' gradient, which moves roundings alone
    for some in itertools.combinations(range(5), 2):
        part = [t.clone().requires_grad_(i in some) for i, t in enumerate(x)]
        got = torch.autograd.grad(W.decay_linear_attention(*part[:4], initial_state=part[4]), [part[i] for i in some], douts)
        for a, i in zip(got, some):
            assert (a.double() - want[i].double()).norm() <= 2 * torch.finfo(dtype).eps * want[i].double().norm(), some
    one = torch.autograd.grad(results[0], leaves, douts[0], retain_graph=True)
    other = torch.autograd.grad(results[1], leaves, douts[1], allow_unused=True)
    for a, b, w in zip(one, other, want):
        total = a.double() if b is None else a.double() + b.double()
        assert (total - w.double()).norm() <= 2 * torch.finfo(dtype).eps * (a.double().norm() + (0 if b is None else b.double().norm()))


def test_rope_gradients_asked_for_one_by_one():
    g = torch.Generator().manual_seed(7)
    q, k = (torch.randn(2, 30, h, 64, generator=g).to(DEV) for h in (4, 2))
    pos = torch.randint(0, 99, (30, 1), generator=g).to(DEV)
    inv, sections = W.axis_frequencies(64, axes=1, device=DEV)
    dq, dk = torch.randn(q.shape, generator=g).to(DEV), torch.randn(k.shape, generator=g).to(DEV)
    leaves = [t.clone().requires_grad_(True) for t in (q, k)]
    out = W.rope_axes(leaves[0], pos, inv, sections, k=leaves[1])
    want = torch.autograd.grad(out, leaves, (dq, dk), retain_graph=True)
    for i in range(2):
        assert torch.equal(torch.autograd.grad(out, leaves[i], (dq, dk), retain_graph=True)[0], want[i])
        part = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, k))]
        got = W.rope_axes(part[0], pos, inv, sections, k=part[1])
        assert torch.equal(torch.autograd.grad(got, part[i], (dq, dk))[0], want[i])
