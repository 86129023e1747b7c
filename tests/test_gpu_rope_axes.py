"""``rope_axes`` against its 64-bit form.

Tolerance, element by element: half a step of the output's type (eps / 2 relative: bf16 2^-8, fp32
2^-24), plus the fp32 part of the rotation: the reduced angle (a fraction of a revolution, rounded to
fp32: 2^-26 of one, 2 pi 2^-26 = 1e-7 rad), the sine and cosine (2 ulp, 2.4e-7), two products and a sum
(3 x 2^-24) on each of the pair's two values, together below 2^-20 (|re| + |im|)."""
import pytest
import torch

from oracle import token as OT
from worldattention_amd import hsa as W
from worldattention_amd import workloads

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _close(got, want, x, what):
    """x: the rotated input, whose pair values bound the fp32 part (its largest pair does, head by head)."""
    half = torch.finfo(got.dtype).eps / 2
    size = 2 * x.detach().double().abs().amax(-1, keepdim=True)
    off = (got.detach().double() - want).abs() - half * 1.01 * want.abs() - 2.0 ** -20 * size
    assert got.shape == want.shape and off.max().item() <= 0, f"{what}: {off.max().item():.3e} over the bound"


def _inputs(b, n, h, hk, d, dtype, sections, seed=0, far=10**6):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, n, h, d, generator=g).to(DEV, dtype)
    k = torch.randn(b, n, hk, d, generator=g).to(DEV, dtype)
    pos = torch.randint(-far, far + 1, (b, n, len(sections)), generator=g).to(DEV)
    inv = torch.cat([10000.0 ** -(torch.arange(s, dtype=torch.float64) / max(s, 1)) for s in sections]).to(DEV)
    return q, k, pos, inv


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,n,h,hk,d,sections", [
    (1, 1, 1, 1, 2, (1,)), (2, 1, 8, 2, 128, (22, 21, 21)), (1, 37, 5, 5, 64, (10, 0, 12)), (3, 130, 12, 3, 96, (16, 32)),
    (2, 9, 3, 1, 80, (5, 7, 3, 4)), (1, 65, 2, 2, 33, (3, 5)), (1, 3, 40, 40, 128, (64,)), (1, 2, 1, 1, 1024, (500, 12))])
def test_rotation_and_gradient(dtype, interleaved, b, n, h, hk, d, sections):
    q, k, pos, inv = _inputs(b, n, h, hk, d, dtype, sections)
    q.requires_grad_(True), k.requires_grad_(True)
    got = W.rope_axes(q, pos, inv, sections, k=k, interleaved=interleaved)
    want = [OT.rope_axes(x, pos, inv, sections, interleaved=interleaved) for x in (q, k)]
    grads = [torch.randn_like(x) for x in got]
    got_d = torch.autograd.grad(got, (q, k), grads)
    want_d = torch.autograd.grad(want, (q, k), [g.double() for g in grads])
    for name, o, w, x in zip("qk", got, want, (q, k)):
        _close(o, w, x, f"{name} rotated")
    # the oracle's gradient was cast to the leaves' dtype by torch: compare with the rotation by -angle
    for name, o, g in zip("qk", got_d, grads):
        _close(o, OT.rope_axes(g, -pos, inv, sections, interleaved=interleaved), g, f"d{name}")
    for o, w in zip(got_d, want_d):
        assert torch.allclose(o.double(), w.double(), rtol=2 * torch.finfo(dtype).eps, atol=2.0 ** -18 * 8)


def test_shared_positions_int32_strides_and_one_tensor():
    """One position row for the batch, int32, channel-last views of other layouts, inv_freq in fp32."""
    q, k, pos, inv = _inputs(2, 21, 4, 2, 128, torch.bfloat16, (22, 21, 21))
    want = OT.rope_axes(q, pos[:1].expand(2, -1, -1), inv, (22, 21, 21))
    got = W.rope_axes(q, pos[0].int(), inv, (22, 21, 21))
    _close(got, want, q, "shared int32 positions")
    bhld = q.transpose(1, 2).contiguous().transpose(1, 2)            # [B, H, L, D] memory
    fused = torch.empty(2, 21, 4 * 128 + 8, device=DEV, dtype=torch.bfloat16)
    inside = fused[..., 3:3 + 512].unflatten(-1, (4, 128))            # rows that start on no 16-byte boundary
    inside.copy_(q)
    last = q.transpose(-1, -2).contiguous().transpose(-1, -2)        # channels not contiguous
    strided_pos = torch.stack([pos, pos + 1], -1)[..., 0]
    for view in (bhld, inside, last, q.expand(2, -1, -1, -1)):
        assert torch.equal(W.rope_axes(view, strided_pos, inv, (22, 21, 21)), W.rope_axes(q, pos, inv, (22, 21, 21)))
    small = 10000.0 ** -(torch.arange(64, dtype=torch.float64, device=DEV) / 64).float()
    _close(W.rope_axes(q, pos[..., :1] % 100, small, (64,)), OT.rope_axes(q, pos[..., :1] % 100, small.double(), (64,)), q,
           "fp32 frequencies")


def test_queries_and_keys_both_copied_for_the_kernel():
    """Both tensors with strided channels, all of one size: neither copy's memory serves the other's output."""
    g = torch.Generator().manual_seed(8)
    pos = torch.randint(0, 1000, (700, 1), generator=g).to(DEV)
    inv, sections = W.axis_frequencies(64, axes=1, device=DEV)
    q, k = (torch.randn(3, 700, 64, 8, generator=g).to(DEV).transpose(2, 3) for _ in range(2))
    for _ in range(3):
        got = W.rope_axes(q, pos, inv, sections, k=k)
        for out, x in zip(got, (q, k)):
            # sine, cosine and two rounded products of fp32
            assert ((out.double() - OT.rope_axes(x, pos, inv, sections)).abs() <= 2.0 ** -20 * x.abs().max()).all()


def test_matches_the_models_own_grid_rope():
    """On a frame x height x width grid with the framework's frequencies it is the 3-D RoPE of its workloads."""
    f, hh, ww, d = 3, 5, 7, 128
    x = torch.randn(1, f * hh * ww, 4, d, device=DEV)
    inv, sections = W.axis_frequencies(d, device=DEV)
    t = torch.arange(f * hh * ww, device=DEV)
    pos = torch.stack([t // (hh * ww) + 18, t // ww % hh, t % ww], -1)
    want = workloads.apply_rope_3d(x.double(), workloads.rope_freqs(64, d).to(DEV), f, hh, ww, 18)
    _close(W.rope_axes(x, pos, inv, sections), want, x, "grid")


def test_far_positions_empty_inputs_and_copied_channels():
    far = 2**31 - 1
    q, _, _, inv = _inputs(1, 4, 2, 1, 64, torch.float32, (16, 8))
    pos = torch.tensor([[far, -far], [0, 0], [1, far], [-far, 3]], device=DEV)
    # 2^31 rad in fp64 is off by 2^-22 / 2, as much again in the product: under the 2^-20 of the bound
    _close(W.rope_axes(q, pos, inv, (16, 8)), OT.rope_axes(q, pos, inv, (16, 8)), q, "far")
    nan = q.clone()
    nan[..., 48:] = float("nan")                                     # copied, and nowhere near the pairs
    got = W.rope_axes(nan, pos, inv, (16, 8))
    assert torch.equal(got[..., :48], W.rope_axes(q, pos, inv, (16, 8))[..., :48]) and got[..., 48:].isnan().all()
    assert torch.equal(W.rope_axes(q, pos * 0, inv, (16, 8)), q)
    for shape in ((0, 4, 2, 64), (1, 0, 2, 64), (1, 4, 0, 64)):
        e = torch.empty(shape, device=DEV)
        out = W.rope_axes(e, torch.zeros(shape[1], 2, dtype=torch.int64, device=DEV), inv, (16, 8), k=e)
        assert out[0].shape == shape and out[1].shape == shape


def test_gradients_of_one_output_broadcast_gradients_and_differences():
    q, k, pos, inv = _inputs(2, 33, 4, 2, 64, torch.float32, (16, 16), far=50)
    q.requires_grad_(True), k.requires_grad_(True)
    oq, ok = W.rope_axes(q, pos, inv, (16, 16), k=k)
    dq, dk = torch.autograd.grad(ok.sum(), (q, k), allow_unused=True, retain_graph=True)  # an expanded gradient, for one tensor
    assert dq is None
    _close(dk, OT.rope_axes(torch.ones_like(k), -pos, inv, (16, 16)), torch.ones_like(k), "dk of a sum")
    # a rotation is linear: f(x + step) - f(x) = f(step) . (the gradient's transpose)
    step, g = torch.randn_like(q), torch.randn_like(oq)
    dq, = torch.autograd.grad(oq, q, g)
    lhs = ((W.rope_axes(q + step, pos, inv, (16, 16)) - oq).double() * g.double()).sum()
    rhs = (dq.double() * step.double()).sum()
    assert abs(lhs - rhs) <= 1e-5 * (step.double().norm() * g.double().norm())
    shared = torch.randn(2, 33, 1, 64, device=DEV, requires_grad=True)   # one head read by four
    W.rope_axes(shared.expand(-1, -1, 4, -1), pos, inv, (16, 16)).backward(g)
    want = OT.rope_axes(g, -pos, inv, (16, 16)).sum(2, keepdim=True)
    assert (shared.grad.double() - want).abs().max() <= 1e-5 * want.abs().max()


def test_other_stream_and_graph_replays():
    q, k, pos, inv = _inputs(1, 50, 4, 2, 128, torch.bfloat16, (22, 21, 21))
    want = W.rope_axes(q, pos, inv, (22, 21, 21), k=k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = W.rope_axes(q, pos, inv, (22, 21, 21), k=k)
        got = [x.clone() for x in got]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = W.rope_axes(q, pos, inv, (22, 21, 21), k=k)
    for _ in range(3):
        q.copy_(torch.randn_like(q)), pos.add_(1)
        graph.replay()
        eager = W.rope_axes(q, pos, inv, (22, 21, 21), k=k)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))
