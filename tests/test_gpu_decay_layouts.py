"""``decay_linear_attention`` on token layouts that ``expand`` and overlapping views make.

The bf16 kernels cut a tile's rows off by the byte range of a buffer descriptor, which needs every row to lie
behind the one before it. A copy of the same values must therefore give the same bits as the view."""
import pytest
import torch

from oracle import token as OT
from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8
H = 2


def _normal(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g).to(DEV, dtype)


def _view(kind, g, b, n, d, dtype):
    """``[b, n, H, d]`` whose tokens share memory: one row for all, rows 8 elements apart, or rows of their own."""
    if kind == "own":
        return _normal(g, b, n, H, d, dtype=dtype)
    if kind == "one row":
        return _normal(g, b, 1, H, d, dtype=dtype).expand(-1, n, -1, -1)
    pitch = 8 * (n - 1) + d
    return _normal(g, b * H * pitch, dtype=dtype).as_strided((b, n, H, d), (H * pitch, 8, pitch, 1))


def _run(x, log_decay, initial, lengths, dout, dfinal):
    leaves = {name: t.detach().requires_grad_(True) for name, t in x.items()}
    log_decay, initial = (t.detach().clone().requires_grad_(True) for t in (log_decay, initial))
    out, final = W.decay_linear_attention(leaves["q"], leaves["k"], leaves["v"], log_decay, initial_state=initial, lengths=lengths)
    grads = torch.autograd.grad((out, final), (*leaves.values(), log_decay, initial), (dout, dfinal))
    return (out.detach(), final.detach(), *grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,lengths", [(33, None), (70, None), (70, (70, 33)), (300, (257, 1))])
@pytest.mark.parametrize("kinds", [("own", "one row", "one row", "own"), ("one row", "own", "own", "one row"),
                                   ("own", "windows", "windows", "own"), ("windows", "own", "windows", "windows")])
def test_tokens_that_share_memory(dtype, d, n, lengths, kinds):
    """Views for q, k, v and the outputs' gradient: the bits of copies, and the final state's fp32 sums (2^-16 of the
    sum of magnitudes: fewer than 2^8 roundings of 2^-24)."""
    g = torch.Generator().manual_seed(n + d)
    b = 2
    x = {name: _view(kind, g, b, n, d, dtype) for name, kind in zip("qkv", kinds)}
    dout = _view(kinds[3], g, b, n, d, dtype)
    log_decay = torch.tensor([0.0, -0.01], device=DEV)
    initial, dfinal = (_normal(g, b, H, d, d, dtype=torch.float32) for _ in range(2))
    if lengths is not None:
        lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = _run(x, log_decay, initial, lengths, dout, dfinal)
    copies = {name: t.clone(memory_format=torch.contiguous_format) for name, t in x.items()}
    want = _run(copies, log_decay, initial, lengths, dout.clone(memory_format=torch.contiguous_format), dfinal)
    for name, a, w in zip(("out", "final", "dq", "dk", "dv", "dlog_decay", "dinitial"), got, want):
        assert torch.equal(a, w), name
    _, exact = OT.decay_linear_attention(copies["q"], copies["k"], copies["v"], log_decay, initial_state=initial, lengths=lengths)
    _, size = OT.decay_linear_attention(copies["q"], copies["k"].abs(), copies["v"].abs(), log_decay, initial_state=initial.abs(),
                                        lengths=lengths)
    assert ((got[1].double() - exact).abs() <= 2.0 ** -16 * size).all()


def test_a_single_token_of_any_stride():
    """One token says nothing about the distance between two: 2^24 elements of it are no reason to refuse."""
    g = torch.Generator().manual_seed(1)
    x = [_normal(g, 1, 1, H, 64) for _ in range(3)]
    pool = torch.zeros(1 << 10, dtype=torch.bfloat16, device=DEV)
    far = []
    for i, t in enumerate(x):
        far.append(pool[i * 256:].as_strided((1, 1, H, 64), (1 << 25, 1 << 24, 64, 1)))
        far[-1].copy_(t)
    log_decay = torch.tensor([-0.5, -0.1], device=DEV)
    got, want = W.decay_linear_attention(*far, log_decay), W.decay_linear_attention(*x, log_decay)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_states_on_any_address():
    """An initial state and a final state's gradient that begin on no 16-byte boundary."""
    g = torch.Generator().manual_seed(2)
    x = {name: _normal(g, 1, 70, H, 64) for name in "qkv"}
    dout = _normal(g, 1, 70, H, 64)
    log_decay = torch.tensor([-0.5, -0.1], device=DEV)
    initial, dfinal = (_normal(g, 1, H, 64, 64, dtype=torch.float32) for _ in range(2))
    odd = []
    for t in (initial, dfinal):
        pool = torch.zeros(t.numel() + 1, device=DEV)
        odd.append(pool[1:].view(t.shape))
        odd[-1].copy_(t)
    want = _run(x, log_decay, initial, None, dout, dfinal)
    leaves = {name: t.detach().clone().requires_grad_(True) for name, t in x.items()}
    decay, state = log_decay.clone().requires_grad_(True), odd[0].requires_grad_(True)
    out, final = W.decay_linear_attention(leaves["q"], leaves["k"], leaves["v"], decay, initial_state=state)
    got = (out.detach(), final.detach(), *torch.autograd.grad((out, final), (*leaves.values(), decay, state), (dout, odd[1])))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
