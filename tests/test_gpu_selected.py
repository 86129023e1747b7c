"""``select_key_blocks``, ``selected_attention`` and ``attend_selected`` against their 64-bit forms.

Choices are equal, ids and counts (scores are fp64 on both sides). Attention, element by element, with
u = 2^-8 (half a step of bf16) and M = softmax-weighted |v|: the weights are rounded once each (u of
every weight): u M, the output's own rounding u |y|, and the fp32 scores: D products of bf16 (2^-24 each
step, D 2^-24 |q||k| scale <= 2^-13 at these sizes) and an exponential: 2^-11 M. The log-sum-exp is of
unrounded weights: 2^-12."""
import math

import pytest
import torch

from oracle import token as OT
from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8


def _cache(b, cap, hk, d, bs, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(b, cap, hk, d, generator=g) + 0.5 * torch.randn(b, -(-cap // bs), hk, d, generator=g).repeat_interleave(bs, 1)[:, :cap]
    v = torch.randn(b, cap, hk, d, generator=g)
    cache = {"k": torch.zeros(b, cap, hk, d, dtype=torch.bfloat16, device=DEV),
             "v": torch.zeros(b, cap, hk, d, dtype=torch.bfloat16, device=DEV)}
    W.kv_append(cache, k.to(DEV).bfloat16(), v.to(DEV).bfloat16(), write_start=0, block_size=bs)
    return cache, g


def _check(q, cache, lens, topk, sink, local, scale=None):
    bs = cache["k_block_sums_block_size"]
    out, lse, chosen = W.attend_selected(q, cache, lens, topk=topk, sink_blocks=sink, local_blocks=local, scale=scale)
    host = [int(x) for x in lens] if isinstance(lens, torch.Tensor) else [lens] * q.shape[0]
    host = [max(0, min(x, cache["k"].shape[1])) for x in host]
    index, num = OT.select_key_blocks(q, cache["k_block_sums"], host, block_size=bs, topk=topk, sink_blocks=sink, local_blocks=local)
    assert torch.equal(chosen.num.cpu(), num)
    assert torch.equal(chosen.index.cpu(), index)
    _check_attention(out, lse, q, cache["k"], cache["v"], index, num, host, bs, scale)
    return out, lse, chosen


def _check_attention(out, lse, q, k, v, index, num, host, bs, scale=None):
    want, want_lse = OT.selected_attention(q, k, v, index, num, host, block_size=bs, scale=scale)
    mag, _ = OT.selected_attention(q, k, v.abs(), index, num, host, block_size=bs, scale=scale)
    assert out.dtype == torch.bfloat16 and lse.dtype == torch.float32
    err = (out.cpu().double() - want).abs()
    assert (err <= U * mag + U * want.abs() + 2.0 ** -11 * mag).all(), (err - U * mag - U * want.abs()).max()
    got = lse.cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want_lse))
    fine = torch.isfinite(want_lse)
    assert ((got - want_lse).abs()[fine] <= 2.0 ** -12).all()
    empty = torch.isinf(want_lse).transpose(1, 2)
    assert (out.cpu()[empty] == 0).all()


@pytest.mark.parametrize("bs", [64, 128])
@pytest.mark.parametrize("b,n,h,hk,d,cap,topk,sink,local", [
    (1, 1, 1, 1, 64, 1, 1, 0, 1), (1, 1, 8, 2, 128, 1000, 4, 1, 2), (3, 1, 12, 12, 128, 2000, 6, 0, 1),
    (2, 5, 8, 1, 64, 1500, 5, 2, 1), (1, 33, 4, 2, 128, 700, 3, 1, 1), (2, 2, 20, 1, 64, 900, 8, 1, 1),
    (1, 1, 48, 1, 128, 3000, 40, 1, 1), (4, 3, 6, 3, 128, 1300, 64, 3, 4), (1, 2, 5, 5, 64, 6000, 16, 1, 2),
    (1, 130, 4, 4, 64, 500, 4, 1, 1), (2, 523, 4, 4, 128, 900, 4, 1, 1), (1, 1101, 8, 4, 64, 1200, 4, 1, 1)])
def test_against_the_oracle(bs, b, n, h, hk, d, cap, topk, sink, local):
    """Ragged lengths: the whole cache, one token, none, around block ends, below the number of queries, past the cache."""
    cache, g = _cache(b, cap, hk, d, bs, seed=cap)
    q = torch.randn(b, n, h, d, generator=g).bfloat16().to(DEV)
    for lens in ([cap, 1, 0, cap + 99], [bs, bs + 1, 2 * bs - 1, -5], [max(1, cap - 1), n - 1, 17, cap // 2]):
        _check(q, cache, torch.tensor(lens[:b], dtype=torch.int32, device=DEV), topk, sink, local)
    _check(q, cache, cap, topk, sink, local, scale=0.3)


@pytest.mark.parametrize("b,hk,d", [(130, 4, 64), (128, 8, 64), (1024, 1, 128), (514, 8, 64)])
def test_many_sequences_of_single_tokens(b, hk, d):
    """Enough key heads that a row, and a choice, gets fewer waves."""
    cache, g = _cache(b, 400, hk, d, 64, seed=b)
    q = torch.randn(b, 1, 2 * hk, d, generator=g).bfloat16().to(DEV)
    lens = torch.randint(0, 420, (b,), generator=g, dtype=torch.int32)
    _check(q, cache, lens.to(DEV), 4, 1, 1)


@pytest.mark.parametrize("nb", [1, 255, 256, 257, 1024, 1025, 4096, 4097, 16384, 16385, 32768])
def test_every_cache_length_the_choice_is_cut_for(nb):
    """The choice alone, at the block counts where its launch changes."""
    g = torch.Generator().manual_seed(nb)
    sums = torch.randn(1, 2, nb, 64, generator=g).to(DEV)
    q = torch.randn(1, 2, 4, 64, generator=g).bfloat16().to(DEV)
    topk = min(24, nb)
    sink = 1 if topk > 1 else 0
    for n_tok in (nb * 64, nb * 64 - 63):
        got = W.select_key_blocks(q, sums, n_tok, block_size=64, topk=topk, sink_blocks=sink)
        index, num = OT.select_key_blocks(q, sums, [n_tok], block_size=64, topk=topk, sink_blocks=sink)
        assert torch.equal(got.num.cpu(), num) and torch.equal(got.index.cpu(), index)


@pytest.mark.parametrize("n,nb", [(1, 1024), (1, 1025), (8, 1024), (9, 1024), (15, 512), (16, 512), (17, 512), (16, 513), (40, 100),
                                  (8, 1000), (8, 1001)])
def test_every_number_of_queries_the_choice_is_cut_for(n, nb):
    """One launch or two, one query tile or several; the first queries before the sequence's first token."""
    g = torch.Generator().manual_seed(n * nb)
    sums = torch.randn(2, 2, nb, 128, generator=g).to(DEV)
    q = torch.randn(2, n, 6, 128, generator=g).bfloat16().to(DEV)
    for lens in ((nb * 64, nb * 32 + 7), (n - 1, 64 * 20), (0, 64 * 9 + 1)):
        kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
        got = W.select_key_blocks(q, sums, kv_len, block_size=64, topk=7, sink_blocks=2, local_blocks=2)
        index, num = OT.select_key_blocks(q, sums, lens, block_size=64, topk=7, sink_blocks=2, local_blocks=2)
        assert torch.equal(got.num.cpu(), num) and torch.equal(got.index.cpu(), index)


@pytest.mark.parametrize("nb", [200, 800, 3000, 9000])
def test_ties_infinities_and_nan_in_the_scores(nb):
    """Equal scores (few distinct values, zeros of both signs), infinite and NaN sums, long runs of ties."""
    g = torch.Generator().manual_seed(nb)
    q = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    q[0, 0, 1] = 2
    sums = torch.zeros(1, 2, nb, 64, device=DEV)
    sums[0, 0, :, 0] = torch.randint(-2, 3, (nb,), generator=g).float().to(DEV)
    sums[0, 1, 5:40:7, 0] = -0.0
    for extra in ({}, {3: math.inf, 70: -math.inf, 150: math.nan, 151: math.nan}):
        for j, x in extra.items():
            sums[0, :, j, 0] = x
        for topk in (2, 3, 31, nb // 2, nb - 1):
            got = W.select_key_blocks(q, sums, nb * 64, block_size=64, topk=topk, sink_blocks=1)
            index, num = OT.select_key_blocks(q, sums, [nb * 64], block_size=64, topk=topk, sink_blocks=1)
            assert torch.equal(got.num.cpu(), num) and torch.equal(got.index.cpu(), index), (topk, extra)


def test_nothing_behind_a_sequence_is_used():
    """NaN and infinities in the cache and the sums behind every sequence's end leave the results' bits."""
    bs, cap = 64, 900
    cache, g = _cache(3, cap, 2, 128, bs, seed=1)
    q = torch.randn(3, 2, 8, 128, generator=g).bfloat16().to(DEV)
    lens = torch.tensor([700, 129, 1], dtype=torch.int32, device=DEV)
    clean = _check(q, cache, lens, 6, 1, 2)
    for b, n in enumerate(lens.tolist()):
        cache["k"][b, n:] = math.nan
        cache["v"][b, n:] = math.inf
        cache["v"][b, n::2] = math.nan
        cache["k_block_sums"][b, :, n // bs:] = math.nan       # the own, partial block's sum is not read either
    dirty = W.attend_selected(q, cache, lens, topk=6, sink_blocks=1, local_blocks=2)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    assert torch.equal(clean[2].index, dirty[2].index) and torch.equal(clean[2].num, dirty[2].num)


def test_any_lists_and_strided_caches():
    """Lists of the caller's own: repeated ids, ids outside the cache, counts outside the list, unordered; a cache that is a
    slice of a larger one with heads outside tokens."""
    g = torch.Generator().manual_seed(8)
    b, n, h, hk, d, cap, bs = 2, 3, 6, 2, 64, 500, 64
    pool = torch.randn(b, hk + 1, cap + 40, 2, d, generator=g).bfloat16().to(DEV)
    k, v = (pool[:, 1:, 13:13 + cap, i].transpose(1, 2) for i in (0, 1))
    q = torch.randn(b, n, d, h, generator=g).bfloat16().to(DEV).transpose(2, 3)      # channels not contiguous
    index = torch.randint(-3, 12, (b, n, hk, 9), generator=g, dtype=torch.int32)
    index[0, 0, 0, :4] = torch.tensor([2**31 - 1, -2**31, 1, 1], dtype=torch.int32)
    num = torch.randint(0, 10, (b, n, hk), generator=g, dtype=torch.int32)
    num[0, 0, 0], num[1, 2, 1], num[1, 1, 0] = 4, -2, 50
    lens = torch.tensor([cap, 200], dtype=torch.int32, device=DEV)
    out, lse = W.selected_attention(q, k, v, index.to(DEV), num.to(DEV), lens, block_size=bs)
    _check_attention(out, lse, q, k, v, index, num.clamp(0, 9), lens.tolist(), bs)


def test_extreme_scores():
    """Scores of +-10^4 and rows whose keys are all equal: the running maximum moves far and stays."""
    bs, cap = 64, 1100
    cache, g = _cache(1, cap, 1, 128, bs, seed=4)
    cache["k"][:, ::3] *= 100
    cache["k"][:, 600:] = cache["k"][:, 600:601]
    q = torch.randn(1, 4, 4, 128, generator=g).bfloat16().to(DEV) * 10
    q[0, 0] = 0
    index = torch.arange(18, dtype=torch.int32).expand(1, 4, 1, 18).contiguous()
    num = torch.full((1, 4, 1), 18, dtype=torch.int32)
    out, lse = W.selected_attention(q, cache["k"], cache["v"], index.to(DEV), num.to(DEV), cap, block_size=bs)
    want, want_lse = OT.selected_attention(q, cache["k"], cache["v"], index, num, [cap], block_size=bs)
    # |scores| reach 2^14: their fp32 error 2^-24 * 2^14 * 8 moves a weight by 2^-7 at most
    mag, _ = OT.selected_attention(q, cache["k"], cache["v"].abs(), index, num, [cap], block_size=bs)
    assert ((out.cpu().double() - want).abs() <= U * mag + U * want.abs() + 2.0 ** -7 * mag).all()
    assert ((lse.cpu().double() - want_lse).abs() <= 2.0 ** -7).all()


@pytest.mark.parametrize("n", [1, 3, 4200])
def test_scores_far_below_zero_are_no_empty_rows(n):
    """All of a row's scores near -10^33 (bf16 reaches 10^38): the largest still gets the weight, whatever number of waves
    and parts a row has."""
    cap, bs = 2048, 64
    g = torch.Generator().manual_seed(12)
    k = torch.zeros(1, cap, 1, 64)
    k[..., 0] = -1e32 * (2 + torch.randperm(cap, generator=g).view(1, cap, 1) / cap)
    k = k.bfloat16()
    v = torch.randn(1, cap, 1, 64, generator=g).bfloat16()
    best = k[0, :, 0, 0].argmax().item()
    k[0, best, 0, 0] = -1e32       # the only one of its value
    q = torch.zeros(1, n, 2, 64, dtype=torch.bfloat16)
    q[..., 0] = 80
    index = torch.arange(32, dtype=torch.int32).expand(1, n, 1, 32).contiguous()
    num = torch.full((1, n, 1), 32, dtype=torch.int32)
    num[0, n // 2:] = best // bs + 1
    # every query's own token lies behind the best one's
    lens = cap + n - 1
    out, lse = W.selected_attention(q.to(DEV), torch.cat((k, k[:, :0].new_full((1, n - 1, 1, 64), -3e38)), 1).to(DEV),
                                    torch.cat((v, v.new_zeros(1, n - 1, 1, 64)), 1).to(DEV), index.to(DEV), num.to(DEV), lens, block_size=bs)
    assert torch.equal(out.cpu(), v[:, best].view(1, 1, 1, 64).expand_as(out))
    want = 80 * k[0, best, 0, 0].double() / 8
    assert ((lse.cpu().double() - want).abs() <= 2.0 ** -20 * want.abs()).all()


def test_long_cache_addresses_past_32_bits():
    """2.2 * 10^9 elements of keys: the chosen blocks lie behind the 32-bit range."""
    cap, bs = 2200 * 1024 // 2, 128
    k = torch.zeros(1, cap, 16, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(3)
    tail = torch.randn(2, 700, 16, 128, generator=g).bfloat16().to(DEV)
    k[0, -700:], v[0, -700:] = tail[0], tail[1]
    q = torch.randn(1, 1, 16, 128, generator=g).bfloat16().to(DEV)
    last = cap // bs
    index = torch.arange(last - 5, last, dtype=torch.int32, device=DEV).expand(1, 1, 16, 5).contiguous()
    num = torch.full((1, 1, 16), 5, dtype=torch.int32, device=DEV)
    got = W.selected_attention(q, k, v, index, num, cap, block_size=bs)
    first = cap - 5 * bs
    small_k, small_v = k[:, first:].contiguous(), v[:, first:].contiguous()
    want = W.selected_attention(q, small_k, small_v, index - (last - 5), num, 5 * bs, block_size=bs)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].any()


def test_repeated_calls_streams_and_graph_replays():
    bs, cap = 64, 3000
    cache, g = _cache(2, cap, 2, 128, bs, seed=6)
    q = torch.randn(2, 1, 8, 128, generator=g).bfloat16().to(DEV)
    lens = torch.tensor([cap, 1234], dtype=torch.int32, device=DEV)
    run = lambda: W.attend_selected(q, cache, lens, topk=32, sink_blocks=1, local_blocks=2)  # noqa: E731
    flat = lambda r: (r[0], r[1], r[2].index, r[2].num)  # noqa: E731
    first, again = flat(run()), flat(run())
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (side, other):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one = flat(run())
    with torch.cuda.stream(other):        # at the same time, each with its own workspace
        two = flat(run())
    for s in (side, other):
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, one, two))
    graphs, held = [], []
    for _ in range(2):                    # two captured graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(flat(run()))
        graphs.append(graph)
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=g).bfloat16().to(DEV))
        lens.sub_(100)
        for graph in graphs:
            graph.replay()
        eager = flat(run())
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) and torch.equal(b, e) for a, b, e in zip(*held, eager)), i


def test_no_queries():
    cache, _ = _cache(1, 100, 2, 64, 64)
    out, lse, chosen = W.attend_selected(torch.zeros(1, 0, 4, 64, device=DEV, dtype=torch.bfloat16), cache, 100, topk=4)
    assert out.shape == (1, 0, 4, 64) and lse.shape == (1, 4, 0) and chosen.index.shape == (1, 0, 2, 4)
