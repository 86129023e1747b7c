"""``decay_linear_attention`` and ``decay_linear_step`` against the recurrence in 64 bits.

Tolerances. Write u for half a step of bf16, 2^-8 relative, and M for what a result would be if every
term of its sum had its absolute value (the oracle on |inputs|). With bf16 tensors a product's operand
is rounded once inside a chunk (the decayed q.k), twice on the way through the running state (the
weighted key, the state itself): at most 2 u M and the square of u, then u |y| for the result's own
rounding: 2.1 u M + u |y|, element by element. Those roundings are independent, so as a whole (2-norms)
the error stays below 1.25 u of the result's norm: three roundings of u / sqrt(3) rms at most, u together,
and what a sum's cancellation adds. fp32 results of bf16 tensors come from operands split in two
(2^-17 relative) and sums of at most 2^7 terms at a time: 2^-16 M. fp32 tensors: products and sums in
fp32, 2^-16 M as well."""
import math

import pytest
import torch

from oracle import token as OT
from worldattention_amd import hsa as W
from worldattention_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8
NAMES = ("q", "k", "v", "log_decay", "initial")


def _inputs(b, n, h, d, dv, dtype, seed=0, initial=True, slow=9.0):
    g = torch.Generator().manual_seed(seed)
    x = {"q": torch.randn(b, n, h, d, generator=g).to(DEV, dtype), "k": torch.randn(b, n, h, d, generator=g).to(DEV, dtype),
         "v": torch.randn(b, n, h, dv, generator=g).to(DEV, dtype),
         "log_decay": -torch.exp2(-torch.rand(h, generator=g) * slow).to(DEV),
         "initial": torch.randn(b, h, d, dv, generator=g).to(DEV) if initial else None}
    grads = torch.randn(b, n, h, dv, generator=g).to(DEV, dtype), torch.randn(b, h, d, dv, generator=g).to(DEV)
    return x, grads


def _all(fn, x, grads, cast=lambda t: t):
    """Results and gradients of ``fn`` as a dict."""
    leaves = {n: cast(t.detach()).clone().requires_grad_(True) for n, t in x.items() if t is not None}
    out, final = fn(leaves["q"], leaves["k"], leaves["v"], leaves["log_decay"], leaves.get("initial"))
    got = torch.autograd.grad((out, final), list(leaves.values()), [g.to(o.dtype) for g, o in zip(grads, (out, final))])
    return {"out": out.detach(), "final": final.detach(), **{"d" + n: t for n, t in zip(leaves, got)}}


def _oracle(x, grads, lengths=None, scale=None):
    f = lambda q, k, v, g, s: OT.decay_linear_attention(q, k, v, g, initial_state=s, lengths=lengths, scale=scale)  # noqa: E731
    want = _all(f, x, grads, torch.Tensor.double)
    size = {n: t if n == "log_decay" or t is None else t.abs() for n, t in x.items()}
    mag = _all(f, size, [t.abs() for t in grads], torch.Tensor.double)
    return want, mag


def _compare(got, want, mag, dtype):
    for name, w in want.items():
        o = got[name].double()
        assert o.shape == w.shape and torch.isfinite(o).all(), name
        rounded = got[name].dtype == torch.bfloat16
        bound = (2.1 * U * mag[name] + U * w.abs() if rounded else 2.0 ** -16 * mag[name]) + 1e-30
        over = ((o - w).abs() / bound).max().item() if o.numel() else 0.0
        assert over <= 1, f"{name}: {over:.2f} of the bound"
        if rounded and w.numel() >= 4096:
            rel = ((o - w).norm() / w.norm()).item()
            assert rel <= 1.25 * U, f"{name}: {rel:.2e} of the norm"
    assert got["out"].dtype == dtype and got["final"].dtype == torch.float32


def _own(lengths=None, scale=None):
    return lambda q, k, v, g, s: W.decay_linear_attention(q, k, v, g, initial_state=s, lengths=lengths, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,n,h,d,dv", [(1, 1, 1, 64, 64), (2, 63, 3, 64, 64), (1, 64, 2, 128, 128), (2, 65, 2, 128, 128),
                                        (1, 130, 1, 128, 128), (3, 200, 2, 64, 64), (1, 700, 2, 128, 128),
                                        (4, 520, 40, 64, 64), (2, 77, 2, 48, 48), (1, 140, 2, 80, 128), (1, 9, 2, 16, 5)])
def test_outputs_and_gradients(dtype, b, n, h, d, dv):
    x, grads = _inputs(b, n, h, d, dv, dtype, seed=n)
    _compare(_all(_own(), x, grads), *_oracle(x, grads), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padded_batch_ignores_what_lies_behind(dtype):
    """Lengths 0, 1, on and around chunk and segment ends, past L; NaN and infinities behind them."""
    n, lengths = 300, torch.tensor([300, 0, 1, 64, 65, 128, 129, 256, 9999, -3], dtype=torch.int32, device=DEV)
    b = lengths.numel()
    x, grads = _inputs(b, n, 2, 64, 64, dtype, seed=5)
    want, mag = _oracle(x, grads, lengths=lengths.clamp(0, n))
    behind = torch.arange(n, device=DEV) >= lengths[:, None]
    for name, bad in (("q", math.inf), ("k", math.nan), ("v", math.nan)):
        x[name][behind] = bad
    grads[0][behind] = math.nan
    got = _all(_own(lengths=lengths), x, grads)
    _compare(got, want, mag, dtype)
    for name in ("out", "dq", "dk", "dv"):
        assert (got[name][behind] == 0).all(), name


def test_decays_of_zero_and_one_and_no_initial_state():
    x, grads = _inputs(2, 150, 4, 64, 64, torch.bfloat16, seed=3, initial=False)
    x["log_decay"] = torch.tensor([0.0, -math.inf, -1e30, -20.0], device=DEV)
    finite = dict(x, log_decay=x["log_decay"].clamp(min=-1e30))
    want, mag = _oracle(finite, grads, scale=0.5)
    _compare(_all(_own(scale=0.5), x, grads), want, mag, torch.bfloat16)
    q, k, v = (x[n][:, :, 1].double() for n in "qkv")
    alone = 0.5 * (q * k).sum(-1, keepdim=True) * v      # a head without memory sees its own token
    out, _ = W.decay_linear_attention(x["q"], x["k"], x["v"], x["log_decay"], scale=0.5)
    assert ((out[:, :, 1].double() - alone).abs() <= 2.1 * U * 0.5 * (q * k).abs().sum(-1, keepdim=True) * v.abs() + U * alone.abs() + 1e-30).all()


def test_gradient_of_the_decays_against_differences():
    x, grads = _inputs(1, 150, 3, 64, 64, torch.float32, seed=9, slow=6.0)
    got = _all(_own(), x, grads)["dlog_decay"].double()
    loss = lambda g: sum((r.double() * w.double()).sum((0, 1, 3) if i == 0 else (0, 2, 3)) for i, (r, w) in enumerate(zip(  # noqa: E731
        OT.decay_linear_attention(x["q"], x["k"], x["v"], g, initial_state=x["initial"]), grads)))
    g0, eps = x["log_decay"].double(), 1e-5
    diff = (loss(g0 + eps) - loss(g0 - eps)) / (2 * eps)
    assert torch.allclose(got, diff, rtol=1e-4, atol=1e-4 * diff.abs().max().item())


def test_strides_shared_heads_and_gradients_of_one_result():
    x, grads = _inputs(2, 140, 4, 64, 64, torch.bfloat16, seed=11)
    bhld = {n: x[n].transpose(1, 2).contiguous().transpose(1, 2) for n in "qkv"}
    wide = torch.zeros(2, 140, 4 * 64 + 3, device=DEV, dtype=torch.bfloat16)
    wide[..., 3:] = x["v"].flatten(2)
    bhld["v"] = wide[..., 3:].unflatten(-1, (4, 64))                       # rows on no 16-byte boundary
    want = W.decay_linear_attention(x["q"], x["k"], x["v"], x["log_decay"], initial_state=x["initial"])
    got = W.decay_linear_attention(bhld["q"], bhld["k"], bhld["v"], x["log_decay"], initial_state=x["initial"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one key and value head for four query heads
    shared = dict(x, k=x["k"][:, :, :1], v=x["v"][:, :, :1])
    wide_heads = lambda f: lambda q, k, v, g, s: f(q, k.expand(-1, -1, 4, -1), v.expand(-1, -1, 4, -1), g, s)  # noqa: E731
    got = _all(wide_heads(_own()), shared, grads)
    f = wide_heads(lambda q, k, v, g, s: OT.decay_linear_attention(q, k, v, g, initial_state=s))
    want = _all(f, shared, grads, torch.Tensor.double)
    size = {n: t if n == "log_decay" else t.abs() for n, t in shared.items()}
    mag = _all(f, size, [t.abs() for t in grads], torch.Tensor.double)
    for name in ("dk", "dv"):      # four rounded gradients, summed and rounded by torch: 1.1 u M more
        mag[name] = mag[name] * 2
    _compare(got, want, mag, torch.bfloat16)
    # the gradient of one result alone; an expanded one
    leaf = x["k"].clone().requires_grad_(True)
    out, final = W.decay_linear_attention(x["q"], leaf, x["v"], x["log_decay"])
    got = torch.autograd.grad(final, leaf, grads[1], retain_graph=True)[0], torch.autograd.grad(out.sum(), leaf)[0]
    one = x["k"].double().requires_grad_(True)
    out, final = OT.decay_linear_attention(x["q"], one, x["v"], x["log_decay"])
    want = torch.autograd.grad(final, one, grads[1].double(), retain_graph=True)[0], torch.autograd.grad(out.sum(), one)[0]
    for a, w in zip(got, want):
        assert ((a.double() - w).norm() / w.norm()).item() <= 1.25 * U


def test_empty_inputs():
    g = torch.full((2,), -0.1, device=DEV)
    s = torch.randn(3, 2, 64, 64, device=DEV)
    e = torch.zeros(3, 0, 2, 64, device=DEV)
    out, final = W.decay_linear_attention(e, e, e, g, initial_state=s)
    assert out.shape == e.shape and torch.equal(final, s) and final.data_ptr() != s.data_ptr()
    out, final = W.decay_linear_attention(e, e, e, g)
    assert not final.any() and final.shape == s.shape
    kept = s.clone()
    assert W.decay_linear_step(e, e, e, g, s).shape == e.shape and torch.equal(kept, s)
    none = torch.zeros(0, 5, 2, 64, device=DEV)
    out, final = W.decay_linear_attention(none, none, none, g)
    assert out.shape == none.shape and final.shape == (0, 2, 64, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,n,h,d,dv", [(1, 1, 1, 1, 1), (3, 1, 5, 64, 64), (2, 1, 12, 128, 128), (2, 5, 3, 80, 96), (1, 3, 2, 33, 7),
                                        (2, 2, 2, 256, 256)])
def test_step(dtype, b, n, h, d, dv):
    """Element by element: the state's update rounds twice in fp32; the output sums D fp32 products: 2^-16 M, then u |y|."""
    x, _ = _inputs(b, n, h, d, dv, dtype, seed=d)
    run = lambda y: OT.decay_linear_attention(y["q"], y["k"], y["v"], y["log_decay"], initial_state=y["initial"])  # noqa: E731
    want, want_s = run(x)
    mag, mag_s = run({m: t if m == "log_decay" else t.abs() for m, t in x.items()})
    pool = torch.full((b + 1, h + 2, d, dv), 7.0, device=DEV)                # the states inside a larger pool
    state = pool[1:, 1:-1]
    state.copy_(x["initial"])
    out = W.decay_linear_step(x["q"], x["k"], x["v"], x["log_decay"], state)
    half = U if dtype == torch.bfloat16 else 0.0
    assert out.dtype == dtype and ((out.double() - want).abs() <= 2.0 ** -16 * mag + half * want.abs()).all()
    assert ((state.double() - want_s).abs() <= 2.0 ** -20 * mag_s).all()
    assert (pool[0] == 7).all() and (pool[:, 0] == 7).all() and (pool[:, -1] == 7).all()


def test_step_with_channels_that_are_not_contiguous():
    """A transposed view, and a single channel whose stride says nothing."""
    for d in (1, 6):
        g = torch.Generator().manual_seed(d)
        q, k, v = (torch.randn(2, 1, d, 5, generator=g).to(DEV).transpose(2, 3) for _ in range(3))
        log_decay = -torch.rand(5, generator=g).to(DEV)
        state = torch.randn(2, 5, d, d, generator=g).to(DEV)
        want, want_s = OT.decay_linear_attention(q, k, v, log_decay, initial_state=state)
        out = W.decay_linear_step(q, k, v, log_decay, state)
        # sums of at most 7 terms below 2^5 in fp32
        assert ((out.double() - want).abs() <= 2.0 ** -15).all() and ((state.double() - want_s).abs() <= 2.0 ** -15).all()


def test_steps_continue_a_prompt():
    x, _ = _inputs(2, 201, 3, 128, 128, torch.bfloat16, seed=21, initial=False)
    want, want_s = OT.decay_linear_attention(x["q"], x["k"], x["v"], x["log_decay"])
    mag, mag_s = OT.decay_linear_attention(x["q"].abs(), x["k"].abs(), x["v"].abs(), x["log_decay"])
    _, state = W.decay_linear_attention(*(x[n][:, :190] for n in "qkv"), x["log_decay"])
    for t in range(190, 201):
        out = W.decay_linear_step(*(x[n][:, t:t + 1] for n in "qkv"), x["log_decay"], state)
        assert ((out[:, 0].double() - want[:, t]).abs() <= 2.0 ** -15 * mag[:, t] + U * want[:, t].abs()).all()
    assert ((state.double() - want_s).abs() <= 2.0 ** -15 * mag_s).all()


def test_repeated_calls_streams_and_graph_replays():
    """Same bits on every call; a captured forward and backward replayed between eager calls; a side stream."""
    x, grads = _inputs(2, 333, 3, 128, 128, torch.bfloat16, seed=31)
    first, again = _all(_own(), x, grads), _all(_own(), x, grads)
    assert all(torch.equal(first[n], again[n]) for n in first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _all(_own(), x, grads)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first[n], other[n]) for n in first)
    leaves = {n: t.clone().requires_grad_(True) for n, t in x.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = W.decay_linear_attention(leaves["q"], leaves["k"], leaves["v"], leaves["log_decay"], initial_state=leaves["initial"])
        held = (*out, *torch.autograd.grad(out, list(leaves.values()), grads))
    for i in range(3):
        fresh, _ = _inputs(2, 333, 3, 128, 128, torch.bfloat16, seed=40 + i)
        with torch.no_grad():
            for n, t in leaves.items():
                t.copy_(fresh[n])
        graph.replay()
        eager = _all(_own(), fresh, grads)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager.values())), i


def test_long_sequences_address_past_32_bits():
    """One head of a tensor whose tokens lie 2^31 elements apart in all."""
    n, pitch = 2100, 1 << 20
    big = torch.empty(n * pitch + 64, dtype=torch.bfloat16, device=DEV)
    view = big.as_strided((1, n, 1, 64), (n * pitch, pitch, 64, 1))
    x, _ = _inputs(1, n, 1, 64, 64, torch.bfloat16, seed=2)
    view.copy_(x["k"])
    want = W.decay_linear_attention(x["q"], x["k"], x["v"], x["log_decay"])
    got = W.decay_linear_attention(x["q"], view, x["v"], x["log_decay"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert _lib.lib().wa_decay_segments(1, n, 1, 0) > 1
