"""The token-by-token operators side by side: captured graphs whose lengths, positions and cache move on, and calls on
several streams at once."""
import pytest
import torch

from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _captured(run):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    return graph, held


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padded_batches_replayed_with_other_lengths(dtype):
    """Two graphs of one padded training call, replayed in turn while the lengths change between 0 and the whole."""
    g = torch.Generator().manual_seed(3)
    b, n, h, d = 3, 400, 2, 64
    x = [torch.randn(b, n, h, d, generator=g).to(DEV, dtype) for _ in range(3)]
    x += [-torch.rand(h, generator=g).to(DEV), torch.randn(b, h, d, d, generator=g).to(DEV)]
    douts = torch.randn(b, n, h, d, generator=g).to(DEV, dtype), torch.randn(b, h, d, d, generator=g).to(DEV)
    lengths = torch.tensor([n, 17, 0], dtype=torch.int32, device=DEV)

    def run(leaves):
        out = W.decay_linear_attention(*leaves[:4], initial_state=leaves[4], lengths=lengths)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, douts))

    eager = lambda: run([t.clone().requires_grad_(True) for t in x])  # noqa: E731
    eager()                                                           # the library is loaded before a capture
    leaves = [[t.clone().requires_grad_(True) for t in x] for _ in range(2)]     # a graph's inputs live as long as it
    graphs = [_captured(lambda own=own: run(own)) for own in leaves]
    for now in ([n, 17, 0], [0, 0, 0], [129, n, 256], [1, 64, n + 5]):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        for graph, _ in graphs:
            graph.replay()
        want = eager()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert all(torch.equal(a, w) for a, w in zip(held, want)), now


def test_a_captured_decoding_step_moves_on():
    """One graph of rotation, selected attention and the recurrent step; position, cache length, cache and state move between
    its replays, eager calls among them."""
    g = torch.Generator().manual_seed(4)
    bs, cap, d = 64, 400, 64
    cache = {name: torch.zeros(1, cap, 2, d, dtype=torch.bfloat16, device=DEV) for name in "kv"}
    tokens = {name: torch.randn(1, 200, hh, d, generator=g).bfloat16().to(DEV) for name, hh in zip("qkv", (4, 2, 2))}
    W.kv_append(cache, tokens["k"][:, :190], tokens["v"][:, :190], write_start=0, block_size=bs)
    inv, sections = W.axis_frequencies(d, axes=1, device=DEV)
    pos, kv_len = torch.tensor([[189]], device=DEV), torch.tensor([190], dtype=torch.int32, device=DEV)
    log_decay, state = torch.tensor([-0.1, -0.2], device=DEV), torch.zeros(1, 2, d, d, device=DEV)
    x = {name: tokens[name][:, 189:190].clone() for name in "qkv"}

    def run():
        q = W.rope_axes(x["q"], pos, inv, sections)
        out, lse, chosen = W.attend_selected(q, cache, kv_len, topk=3)
        return q, out, lse, chosen.index, W.decay_linear_step(x["k"], x["k"], x["v"], log_decay, state)

    run()
    state.zero_()
    graph, held = _captured(run)
    for t in range(190, 196):
        W.kv_append(cache, tokens["k"][:, t:t + 1], tokens["v"][:, t:t + 1], write_start=t, block_size=bs)
        for name in "qkv":
            x[name].copy_(tokens[name][:, t:t + 1])
        pos.fill_(t), kv_len.fill_(t + 1)
        before = state.clone()
        graph.replay()
        after = state.clone()
        state.copy_(before)
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(held, want)) and torch.equal(state, after), t


def test_training_calls_on_two_streams_at_once():
    g = torch.Generator().manual_seed(5)
    x = [torch.randn(2, 700, 3, 128, generator=g).bfloat16().to(DEV) for _ in range(3)]
    x += [-torch.rand(3, generator=g).to(DEV), torch.randn(2, 3, 128, 128, generator=g).to(DEV)]
    dout = torch.randn(2, 700, 3, 128, generator=g).bfloat16().to(DEV)

    def run():
        leaves = [t.clone().requires_grad_(True) for t in x]
        out, final = W.decay_linear_attention(*leaves[:4], initial_state=leaves[4])
        return [out.detach(), final.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 3:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for r in got:
        assert all(torch.equal(a, w) for a, w in zip(r, want))
