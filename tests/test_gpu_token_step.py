"""The token-by-token operators together, as a model with both kinds of heads runs them: a prompt of mixed tokens, then
single tokens. Every stage is checked against its 64-bit form on what the stage was given (rotation: half a step of
bf16 of the result and 2^-20 of the pair; choice: equal; attention and decayed attention: the bounds of their own
tests), the cache and the states against what the stages before must have left."""
import pytest
import torch

from oracle import token as OT
from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8
SPARSE, KV, LINEAR, D, BS = 8, 2, 3, 64, 64


def _rotated(x, pos, inv, sections):
    want = OT.rope_axes(x, pos, inv, sections)
    return want, U * want.abs() + 2.0 ** -20 * x.double().abs().amax(-1, keepdim=True)


def _close(got, want, bound):
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() - bound).max()


class _Layer:
    """Sparse heads over a cache, linear heads over a state; one call for the tokens that arrive."""

    def __init__(self, batch, cap):
        self.cache = {n: torch.zeros(batch, cap, KV, D, dtype=torch.bfloat16, device=DEV) for n in ("k", "v")}
        self.inv, self.sections = W.axis_frequencies(D, device=DEV)
        self.log_decay = -torch.exp2(-torch.arange(1, LINEAR + 1).float()).to(DEV)
        self.state, self.at = None, 0

    def __call__(self, x, pos):
        n = pos.shape[0]
        q, k = W.rope_axes(x["q"], pos, self.inv, self.sections, k=x["k"])
        W.kv_append(self.cache, k, x["v"], write_start=self.at, block_size=BS)
        self.at += n
        sparse, lse, chosen = W.attend_selected(q, self.cache, self.at, topk=4, sink_blocks=1, local_blocks=1)
        before = None if self.state is None else self.state.clone()
        if n == 1:
            linear = W.decay_linear_step(x["lq"], x["lk"], x["lv"], self.log_decay, self.state)
        else:
            linear, self.state = W.decay_linear_attention(x["lq"], x["lk"], x["lv"], self.log_decay, initial_state=self.state)
        return dict(q=q, k=k, sparse=sparse, lse=lse, chosen=chosen, linear=linear, before=before)


def _tokens(batch, n, g):
    heads = dict(q=SPARSE, k=KV, v=KV, lq=LINEAR, lk=LINEAR, lv=LINEAR)
    return {name: torch.randn(batch, n, h, D, generator=g).bfloat16().to(DEV) for name, h in heads.items()}


def _check(layer, x, pos, r, written):
    batch, n = x["q"].shape[:2]
    for name in "qk":
        _close(r[name], *_rotated(x[name], pos, layer.inv, layer.sections))
    written["k"].append(r["k"])
    written["v"].append(x["v"])
    for name in "kv":
        assert torch.equal(layer.cache[name][:, :layer.at], torch.cat(written[name], 1)) and not layer.cache[name][:, layer.at:].any()
    lens = [layer.at] * batch
    index, num = OT.select_key_blocks(r["q"], layer.cache["k_block_sums"], lens, block_size=BS, topk=4)
    assert torch.equal(r["chosen"].index.cpu(), index) and torch.equal(r["chosen"].num.cpu(), num)
    args = (layer.cache["k"], index, num, lens)
    want, want_lse = OT.selected_attention(r["q"], layer.cache["k"], layer.cache["v"], *args[1:], block_size=BS)
    mag, _ = OT.selected_attention(r["q"], layer.cache["k"], layer.cache["v"].abs(), *args[1:], block_size=BS)
    _close(r["sparse"].cpu(), want, (U + 2.0 ** -11) * mag + U * want.abs())
    _close(r["lse"].cpu(), want_lse, 2.0 ** -12)
    want, want_s = OT.decay_linear_attention(x["lq"], x["lk"], x["lv"], layer.log_decay, initial_state=r["before"])
    mag, mag_s = OT.decay_linear_attention(x["lq"].abs(), x["lk"].abs(), x["lv"].abs(), layer.log_decay,
                                           initial_state=None if r["before"] is None else r["before"].abs())
    _close(r["linear"], want, 2.1 * U * mag + U * want.abs())
    _close(layer.state, want_s, 2.0 ** -15 * mag_s)


def test_a_prompt_of_mixed_tokens_then_single_ones():
    """A 3-D grid of video tokens and a run of text behind it (all axes equal), then text tokens one at a time, across
    the end of a block; twice, with the same bits."""
    batch, prompt = 2, 4 * 6 * 10 + 10
    grid = torch.stack(torch.meshgrid(torch.arange(4), torch.arange(6), torch.arange(10), indexing="ij"), -1).view(-1, 3)
    text = (torch.arange(40) + 11)[:, None].expand(-1, 3)
    pos = torch.cat((grid, text)).to(DEV)
    runs = []
    for check in (True, False):
        g = torch.Generator().manual_seed(5)
        layer, written, outs = _Layer(batch, 400), {"k": [], "v": []}, []
        first = 0
        for n in [prompt] + [1] * 9:
            x = _tokens(batch, n, g)
            r = layer(x, pos[first:first + n])
            if check:
                _check(layer, x, pos[first:first + n], r, written)
            outs += [r["sparse"], r["lse"], r["linear"]]
            first += n
        runs.append(outs + [layer.state])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_training_step_through_rotation_and_decay():
    """Rotated queries and keys into decayed attention: gradients of the whole chain against fp64's (the rotation rounds its
    results and gradients to bf16 once each, so 2-norms differ by at most 3 u of the gradient's)."""
    g = torch.Generator().manual_seed(9)
    n = 150
    inv, sections = W.axis_frequencies(D, axes=2, device=DEV)
    pos = torch.stack((torch.arange(n) // 10, torch.arange(n) % 10), -1).to(DEV)
    x = {name: torch.randn(2, n, LINEAR, D, generator=g).bfloat16().to(DEV) for name in "qkv"}
    x["g"] = -torch.exp2(-torch.arange(1, LINEAR + 1).float()).to(DEV)
    dout = torch.randn(2, n, LINEAR, D, generator=g).bfloat16().to(DEV)

    def run(rope, attend, cast):
        leaves = {name: cast(t).clone().requires_grad_(True) for name, t in x.items()}
        q, k = rope(leaves["q"], leaves["k"])
        out = attend(q, k, leaves["v"], leaves["g"])[0]
        return [out.detach(), *torch.autograd.grad(out, list(leaves.values()), dout.to(out.dtype))]

    got = run(lambda q, k: W.rope_axes(q, pos, inv, sections, k=k), W.decay_linear_attention, lambda t: t)
    want = run(lambda q, k: [OT.rope_axes(t, pos, inv, sections) for t in (q, k)], OT.decay_linear_attention, torch.Tensor.double)
    for a, b in zip(got, want):
        assert ((a.double() - b).norm() <= 3 * U * b.norm()).item()
