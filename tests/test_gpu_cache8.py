"""The 8-bit cache and the attention over it against their 64-bit forms.

Codes, scales and read values are exact: equal. Block sums of int8 codes are exact too (whole numbers below 2^24 times a power of two);
those of e4m3 codes are fp32 sums of 128 numbers: 128 2^-24 of their magnitudes. Attention, with u = 2^-8 (half a step of bf16) and M the softmax-weighted |v|:
weights times a power of two are rounded once (u M), the output once (u |y|), and scores are fp32 sums of D exact products, bent by a few
2^-24 of the cap and of biases of at most 2^10: weights within 2^-11, the log-sum-exp 2^-12 and 2^-22 of its magnitude."""
import math

import pytest
import torch

from oracle import cache8 as OC
from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8
TYPES = [torch.int8, torch.float8_e4m3fn]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _tokens(g, b, n, hk, d, dtype=torch.bfloat16):
    size = torch.exp2(2 * torch.randn(hk, d, generator=g))
    return (torch.randn(b, n, hk, d, generator=g) * size * torch.exp2(torch.randn(b, n, 1, 1, generator=g))).to(dtype).to(DEV)


def _mirror(cache):
    dtype, bs = cache["k"].dtype, cache["k_block_sums_block_size"]
    return {x: OC.Cache(cache[x].cpu().float(), cache[x + "_scale"], bs, dtype) for x in "kv"}


def _same(cache, mirror, sums=()):
    for x in "kv":
        assert torch.equal(cache[x + "_scale"].double().cpu().nan_to_num(-1.0), mirror[x].scale.nan_to_num(-1.0)), x
        assert torch.equal(cache[x].cpu().float().double(), mirror[x].codes), x
    for (b, h, j), want in dict(sums).items():
        got = cache["k_block_sums"][b, h, j].double().cpu()
        bs = cache["k_block_sums_block_size"]
        rows = mirror["k"].values()[b, j * bs: (j + 1) * bs, h].abs().sum(0)
        off = 0.0 if cache["k"].dtype is torch.int8 else 128 * 2.0 ** -24
        want = want.float().double()       # two keys of 3.4e38 add up to more than fp32 holds: infinite in fp32, whatever the order
        same_inf = torch.isinf(want) & (got == want)
        got, want = torch.where(same_inf, 0.0, got), torch.where(same_inf, 0.0, want)
        assert torch.equal(got.isnan(), want.isnan()) and ((got - want).abs() <= off * rows)[~want.isnan()].all(), (b, h, j)


def _append(cache, mirror, k, v, start, lengths=None):
    b, n = k.shape[:2]
    starts = start if isinstance(start, list) else [start] * b
    counts = [n] * b if lengths is None else lengths
    W.kv_append_8bit(cache, k, v, _i32(start) if isinstance(start, list) else start, lengths=None if lengths is None else _i32(lengths))
    sums = mirror["k"].append(k, starts, counts)
    mirror["v"].append(v, starts, counts)
    _same(cache, mirror, sums)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,bs,src", [(64, 64, torch.bfloat16), (128, 64, torch.float32), (64, 128, torch.float32), (128, 128, torch.bfloat16)])
def test_written_as_defined(dtype, d, bs, src):
    """Prompts, single tokens whose scales grow and do not, drafts taken back, ragged batches, places of their own."""
    b, cap, hk = 3, 333, 2
    g = torch.Generator().manual_seed(d + bs)
    cache = W.new_cache_8bit(b, cap, hk, d, block_size=bs, dtype=dtype)
    mirror = _mirror(cache)
    new = lambda n: (_tokens(g, b, n, hk, d, src), _tokens(g, b, n, hk, d, src))  # noqa: E731
    _append(cache, mirror, *new(150), 0)
    for t in range(150, 153):
        _append(cache, mirror, *new(1), t)
    _append(cache, mirror, *new(5), [153, 10, 64])
    _append(cache, mirror, *new(9), [140, 128, 63])                 # over tokens that were there
    _append(cache, mirror, *new(130), [190, 200, 203], [130, 0, 77])
    _append(cache, mirror, *new(4), [330, -1, 329], [4, 4, 99])      # the first two do not fit: left as they are
    _append(cache, mirror, *new(cap), 0)
    small = [x * 2.0 ** -9 for x in new(40)]                        # a block begun anew takes a smaller scale
    _append(cache, mirror, *small, 128)
    _append(cache, mirror, *[x * 2.0 ** -9 for x in new(20)], 168)   # ... one behind larger tokens keeps theirs


@pytest.mark.parametrize("dtype", TYPES)
def test_single_tokens_one_after_the_other(dtype):
    """A block that grows token by token: within a step of its scale in int8 of what was written."""
    b, cap, hk, d = 2, 130, 1, 64
    g = torch.Generator().manual_seed(3)
    cache = W.new_cache_8bit(b, cap, hk, d, dtype=dtype)
    mirror = _mirror(cache)
    k, v = _tokens(g, b, cap, hk, d), _tokens(g, b, cap, hk, d)
    for t in range(cap):
        _append(cache, mirror, k[:, t:t + 1], v[:, t:t + 1], t)
    got, _ = W.kv_read_8bit(cache, 0, cap, dtype=torch.float32)
    if dtype is torch.int8:
        step = cache["k_scale"].repeat_interleave(64, 2)[:, :, :cap].transpose(1, 2)[..., None]
        assert ((got - k.float()).abs() < step).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_every_value_that_a_code_has(dtype):
    """Ties, the largest and smallest codes, scales at both ends, zeros, values below fp32's normal numbers."""
    d, n = 128, 128
    most = OC.LARGEST[dtype]
    steps = torch.arange(-2 * int(most), 2 * int(most) + 1).float() / 2
    if dtype is not torch.int8:
        steps = torch.cat((steps, steps * 2.0 ** -9, torch.arange(-64, 65) * 2.0 ** -12, torch.arange(-64, 65) * 2.0 ** -6))
    fill = torch.zeros(-(-steps.numel() // (n * d)) * n * d)
    fill[:steps.numel()] = steps
    rows = fill.view(-1, n, 1, d)
    for power in (0, 40, -60, 100, -126, -140):
        x = (rows.double() * 2.0 ** power).float().to(DEV)
        cache = W.new_cache_8bit(x.shape[0], n, 1, d, block_size=128, dtype=dtype)
        _append(cache, _mirror(cache), x, -x, 0)
    for edge in (most * 2.0 ** 3, most * 2.0 ** 3 * (1 + 2.0 ** -20), 2.0 ** -126 * most, 2.0 ** -149, 3.4028234e38):
        x = torch.full((1, 2, 1, d), edge, device=DEV)
        cache = W.new_cache_8bit(1, n, 1, d, dtype=dtype)
        _append(cache, _mirror(cache), x, -x, 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_value_that_is_not_finite_shows_in_its_block(dtype):
    g = torch.Generator().manual_seed(4)
    cache = W.new_cache_8bit(1, 200, 2, 64, dtype=dtype)
    mirror = _mirror(cache)
    k, v = _tokens(g, 1, 200, 2, 64), _tokens(g, 1, 200, 2, 64)
    k[0, 70, 1, 5], v[0, 10, 0, 0], v[0, 199, 1, 63] = math.inf, math.nan, -math.inf
    _append(cache, mirror, k[:, :100], v[:, :100], 0)
    _append(cache, mirror, k[:, 100:], v[:, 100:], 100)
    got_k, got_v = W.kv_read_8bit(cache, 0, 200)
    bad = got_k.isnan().all(-1)[0]
    assert bad[64:128, 1].all() and not bad[:64].any() and not bad[:, 0].any() and not bad[128:].any()
    bad = got_v.isnan().all(-1)[0]
    assert bad[:64, 0].all() and bad[192:, 1].all() and not bad[64:, 0].any() and not bad[:192, 1].any()
    _append(cache, mirror, *(torch.ones(1, 64, 2, 64, device=DEV),) * 2, 64)   # begun anew
    assert W.kv_read_8bit(cache, 64, 64)[0].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,bs", [(64, 128), (128, 64)])
def test_read_back(dtype, d, bs):
    b, cap, hk = 3, 300, 5
    g = torch.Generator().manual_seed(6)
    cache = W.new_cache_8bit(b, cap, hk, d, block_size=bs, dtype=dtype)
    mirror = _mirror(cache)
    _append(cache, mirror, _tokens(g, b, 290, hk, d), _tokens(g, b, 290, hk, d), 0)
    for start, n in ((0, cap), (17, 1), (63, 130), ([0, 5, 250], 50), ([-3, 299, 400], 7)):
        starts = start if isinstance(start, list) else [start] * b
        for out in (torch.bfloat16, torch.float32):
            got = W.kv_read_8bit(cache, _i32(start) if isinstance(start, list) else start, n, dtype=out)
            for x, y in zip("kv", got):
                want = torch.zeros(b, n, hk, d, dtype=torch.float64)
                for i, s in enumerate(starts):
                    for t in range(n):
                        if 0 <= s + t < cap:
                            want[i, t] = mirror[x].values()[i, s + t]
                assert y.dtype is out and torch.equal(y.cpu().double(), want)
    assert W.kv_read_8bit(cache, 0, 0)[0].shape == (b, 0, hk, d)


def _filled(b, cap, hk, d, bs, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    cache = W.new_cache_8bit(b, cap, hk, d, block_size=bs, dtype=dtype)
    k, v = (torch.randn(b, cap, hk, d, generator=g).to(DEV) for _ in range(2))
    W.kv_append_8bit(cache, k, v, 0)
    return cache, g


def _check_attention(got, q, cache, lens, **kw):
    k, v = W.kv_read_8bit(cache, 0, cache["k"].shape[1], dtype=torch.float32)
    bs = cache["k_block_sums_block_size"]
    if "chosen" in kw:
        kw["chosen"] = [t.cpu() for t in kw["chosen"]]
    want, want_lse = OC.attend(q, k, v, lens, block_size=bs, **kw)
    mag, _ = OC.attend(q, k, v.abs(), lens, block_size=bs, **kw)
    out, lse = got[0].cpu().double(), got[1].cpu().double()
    err = (out - want).abs()
    assert (err <= U * mag + U * want.abs() + 2.0 ** -11 * mag).all(), (err - U * mag - U * want.abs()).max()
    fine = torch.isfinite(want_lse)
    assert torch.equal(torch.isinf(lse), ~fine)
    assert ((lse - want_lse).abs()[fine] <= 2.0 ** -12 + 2.0 ** -22 * want_lse.abs()[fine]).all()
    assert (out.transpose(1, 2)[~fine] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,n,h,hk,d,cap,bs,kw", [
    (1, 1, 1, 1, 64, 1, 64, {}), (3, 1, 8, 2, 128, 700, 64, {}), (2, 1, 20, 1, 64, 300, 128, {}), (4, 3, 6, 3, 128, 260, 64, {}),
    (2, 5, 8, 1, 64, 500, 128, dict(cap=9.0)), (1, 16, 4, 1, 128, 333, 64, {}), (2, 9, 7, 7, 64, 200, 64, dict(window=50, sink=3)),
    (1, 1, 48, 1, 128, 900, 64, dict(window=200)), (2, 2, 8, 4, 128, 600, 64, dict(window=90, sink=70)), (2, 33, 2, 1, 64, 400, 64, dict(cap=3.0)),
    (2, 70, 4, 2, 128, 400, 64, dict(window=120, sink=10, cap=5.0)), (2, 140, 4, 2, 128, 400, 64, dict(window=120, sink=10, cap=5.0)),
    (1, 100, 2, 2, 64, 140, 128, {}), (1, 270, 2, 2, 64, 300, 128, {}), (3, 131, 6, 3, 128, 200, 64, dict(window=33)), (1, 1, 4, 2, 64, 5000, 64, {})])
def test_attention_against_the_definition(dtype, b, n, h, hk, d, cap, bs, kw):
    """Ragged lengths: the whole cache, one token, none, around tile and block ends, below the number of queries, past the cache."""
    cache, g = _filled(b, cap, hk, d, bs, dtype, seed=cap)
    q = torch.randn(b, n, h, d, generator=g).bfloat16().to(DEV)
    slopes = (torch.rand(h, generator=g) * 0.2).to(DEV)
    for lens in ([cap, 1, 0, cap + 99], [bs, bs + 1, 33, -5], [max(1, cap - 1), n - 1, 17, cap // 2]):
        _check_attention(W.attend_8bit(q, cache, _i32(lens[:b]), **kw), q, cache, lens[:b], **kw)
    more = dict(kw, scale=0.3, slopes=slopes)
    _check_attention(W.attend_8bit(q, cache, cap, **more), q, cache, [cap] * b, **more)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,bs", [(64, 128), (128, 64)])
def test_chosen_blocks(dtype, d, bs):
    """A choice from the cache's sums, and lists of the caller's own: repeated ids, ids without seen tokens, counts outside the list."""
    b, n, h, hk, cap = 2, 3, 6, 2, 900
    cache, g = _filled(b, cap, hk, d, bs, dtype, seed=7)
    q = torch.randn(b, n, h, d, generator=g).bfloat16().to(DEV)
    for lens in ([cap, 333], [bs + 1, 2], [0, cap + 5]):
        chosen = W.select_key_blocks(q, cache["k_block_sums"], _i32(lens), block_size=bs, topk=5)
        _check_attention(W.attend_8bit(q, cache, _i32(lens), chosen=chosen, cap=20.0), q, cache, lens, chosen=chosen, cap=20.0)
        index = torch.randint(-2, cap // bs + 3, (b, n, hk, 40), generator=g, dtype=torch.int32).to(DEV)
        num = torch.randint(-1, 41, (b, n, hk), generator=g, dtype=torch.int32).to(DEV)
        lists = W.BlockSelection(index, num)
        _check_attention(W.attend_8bit(q, cache, _i32(lens), chosen=lists), q, cache, lens, chosen=lists)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,kw", [(2, dict(window=60, sink=5)), (70, dict(window=60, sink=5)), (140, dict(window=60, sink=5)), (2, {}), (70, {}), (140, {})])
def test_nothing_behind_a_sequence_is_used(dtype, n, kw):
    cap = 400
    cache, g = _filled(2, cap, 2, 64, 64, dtype, seed=8)
    q = torch.randn(2, n, 4, 64, generator=g).bfloat16().to(DEV)
    lens = [301, 65]
    clean = W.attend_8bit(q, cache, _i32(lens), **kw)
    for b, x in enumerate(lens):
        cache["k"][b, x:].view(torch.uint8).fill_(127)     # NaN in e4m3
        cache["v"][b, x:].view(torch.uint8).fill_(255)
        for t in ("k_scale", "v_scale"):
            cache[t][b, :, -(-x // 64):] = math.nan
    dirty = W.attend_8bit(q, cache, _i32(lens), **kw)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


def test_a_block_that_is_not_finite_reaches_those_who_see_it():
    cache, g = _filled(1, 200, 1, 64, 64, torch.int8, seed=9)
    cache["v_scale"][0, 0, 2] = math.nan
    q = torch.randn(1, 4, 2, 64, generator=g).bfloat16().to(DEV)
    out, lse = W.attend_8bit(q, cache, 130)     # queries at 126, 127 (block 1), 128, 129 (block 2)
    assert out[0, :2].isfinite().all() and out[0, 2:].isnan().all() and lse.isfinite().all()


@pytest.mark.parametrize("n", [1, 65, 130])
def test_any_strides_of_queries(n):
    cache, g = _filled(2, 300, 2, 64, 64, torch.int8, seed=10)
    wide = torch.randn(2, 4, n + 3, 80, generator=g).bfloat16().to(DEV)
    q = wide[..., 3:67].transpose(1, 2)[:, 2:2 + n]
    got, want = W.attend_8bit(q, cache, 290), W.attend_8bit(q.contiguous(), cache, 290)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = q[:, :1].expand(2, n, 4, 64)
    assert torch.equal(W.attend_8bit(one, cache, 290)[0], W.attend_8bit(one.contiguous(), cache, 290)[0])
    k = torch.randn(2, 2, 9, 72, generator=g).bfloat16().to(DEV)[..., 5:69].transpose(1, 2)
    other = {x: y.clone() if isinstance(y, torch.Tensor) else y for x, y in cache.items()}
    W.kv_append_8bit(cache, k, k, 100)
    W.kv_append_8bit(other, k.contiguous(), k.contiguous(), 100)
    assert all(torch.equal(cache[x].view(torch.uint8), other[x].view(torch.uint8)) for x in ("k", "v"))


def test_both_ways_agree():
    """The same queries a few at a time over the codes, and all at once over the values read back."""
    cache, g = _filled(2, 500, 2, 128, 64, torch.float8_e4m3fn, seed=12)
    q = torch.randn(2, 144, 4, 128, generator=g).bfloat16().to(DEV)
    slopes = torch.tensor([0.1, 0.02, 0.3, 0.0], device=DEV)
    kw = dict(cap=8.0, slopes=slopes, window=100, sink=4)
    whole, lse = W.attend_8bit(q, cache, _i32([500, 120]), **kw)
    for i in range(0, 144, 48):
        part, part_lse = W.attend_8bit(q[:, i:i + 48], cache, _i32([500 - 96 + i, 120 - 96 + i]), **kw)
        assert ((part - whole[:, i:i + 48]).abs().float() <= 2.0 ** -5).all()      # values of about 1: two roundings to bf16 of a few weights each
        same = lse[:, :, i:i + 48]
        none = torch.isinf(same)      # queries before the first token, in both
        assert torch.equal(none, torch.isinf(part_lse)) and ((part_lse - same).abs()[~none] <= 2.0 ** -10).all()


def test_a_decoding_step_captured():
    """Append, attend and read in a graph with device positions, replayed between eager work; a second graph beside it."""
    b, cap, hk, d = 2, 300, 2, 64
    sets = []
    for seed in (1, 2):
        cache, g = _filled(b, cap, hk, d, 64, torch.int8, seed=seed)
        k, v, q = (torch.randn(b, 1, x, d, generator=g).bfloat16().to(DEV) for x in (hk, hk, 4))
        pos = _i32([100, 63 + seed])

        def step(cache=cache, k=k, v=v, q=q, pos=pos):
            W.kv_append_8bit(cache, k, v, pos)
            return (*W.attend_8bit(q, cache, pos + 1, cap=30.0), *W.kv_read_8bit(cache, pos, 1))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        sets.append((graph, got, step, cache, pos, q))
    for turn in range(4):
        for graph, got, step, cache, pos, q in sets:
            pos += 1
            q.mul_(-1.5)
            before = {x: y.clone() if isinstance(y, torch.Tensor) else y for x, y in cache.items()}
            graph.replay()
            torch.cuda.synchronize()
            want = step(cache=before)
            assert all(torch.equal(x, y) for x, y in zip(got, want)), turn
            assert all(torch.equal(cache[x].view(torch.uint8), before[x].view(torch.uint8)) for x in ("k", "v", "k_scale", "k_block_sums"))


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_selected_on_an_8bit_cache(dtype):
    """The choice and the attention in one call, with lengths past the cache too."""
    cache, g = _filled(2, 700, 2, 128, 64, dtype, seed=14)
    q = torch.randn(2, 3, 8, 128, generator=g).bfloat16().to(DEV)
    for lens in ([700, 130], [705, 2]):
        out, lse, chosen = W.attend_selected(q, cache, _i32(lens), topk=4, local_blocks=2)
        want = W.select_key_blocks(q, cache["k_block_sums"], _i32([min(x, 700) for x in lens]), block_size=64, topk=4, local_blocks=2)
        assert torch.equal(chosen.index, want.index) and torch.equal(chosen.num, want.num)
        _check_attention((out, lse), q, cache, lens, chosen=chosen)
    with pytest.raises(ValueError, match="scale must be above 0"):
        W.attend_selected(q, cache, 700, topk=4, scale=-1.0)


def test_a_cache_whose_offsets_pass_32_bits():
    """Codes behind 2^31 bytes and 2^32: written, read and attended to at the far end, alone and as a chunk."""
    cap, hk, d = (1 << 25) // 8 + 300, 8, 128
    g = torch.Generator().manual_seed(15)
    cache = W.new_cache_8bit(1, cap, hk, d)
    n = 200
    k, v = (torch.randn(1, n, hk, d, generator=g).bfloat16().to(DEV) for _ in range(2))
    start = cap - n - 11
    W.kv_append_8bit(cache, k, v, _i32([start]))
    first = start // 64 * 64
    small = W.new_cache_8bit(1, cap - first, hk, d)
    W.kv_append_8bit(small, k, v, start - first)
    for x, y in zip(W.kv_read_8bit(cache, first, cap - first), W.kv_read_8bit(small, 0, cap - first)):
        assert torch.equal(x, y)
    for rows in (2, 80):
        q = torch.randn(1, rows, hk, d, generator=g).bfloat16().to(DEV)
        far = W.attend_8bit(q, cache, _i32([start + n]), window=64)
        near = W.attend_8bit(q, small, start - first + n, window=64)
        assert torch.equal(far[1], near[1]) or (far[1] - near[1]).abs().max() <= 2.0 ** -10
        assert ((far[0] - near[0]).abs().float() <= 2.0 ** -5).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,h", [(1, 17), (4, 8), (8, 8), (16, 4), (64, 1), (65, 1)])
def test_every_number_of_rows(dtype, d, n, h):
    """Units of one, two and four row tiles, full and not, several of them, and the chunk."""
    cache, g = _filled(1, 310, 1, d, 64, dtype, seed=n * h)
    q = torch.randn(1, n, h, d, generator=g).bfloat16().to(DEV)
    for kw in ({}, dict(window=40, sink=35, cap=4.0)):
        _check_attention(W.attend_8bit(q, cache, 301, **kw), q, cache, [301], **kw)


@pytest.mark.parametrize("b,n,h,hk,d,cap,kw", [
    (2, 1, 4, 2, 128, 4000, {}), (37, 1, 4, 2, 64, 3000, {}), (37, 3, 10, 1, 128, 3000, dict(window=1500, sink=70, cap=9.0)), (5, 2, 21, 3, 64, 2900, {}),
    (256, 1, 2, 1, 64, 900, dict(window=500)), (257, 1, 2, 1, 64, 900, {}), (9, 8, 8, 1, 128, 2500, {}), (3, 1, 16, 16, 64, 2048, {})])
def test_ragged_sequences(b, n, h, hk, d, cap, kw):
    """Tiles shared along all sequences: none, one, the cache's whole length and more, and many in a row that see nothing."""
    cache, g = _filled(b, cap, hk, d, 64, torch.int8, seed=b + n)
    q = torch.randn(b, n, h, d, generator=g).bfloat16().to(DEV)
    lens = torch.randint(0, cap + 1, (b,), generator=g).tolist()
    some = [0, cap + 5, 1, cap][:b]
    for lens in (lens, some + [0] * (b - len(some)), [0] * (b - 1) + [cap], [0] * b, [cap] * b, [-3, 31] + [33] * (b - 2)):
        _check_attention(W.attend_8bit(q, cache, _i32(lens), **kw), q, cache, [min(max(x, 0), cap) for x in lens], **kw)


@pytest.mark.parametrize("n,h,hk", [(127, 1, 1), (128, 2, 2), (129, 1, 1), (64, 8, 2), (65, 8, 2), (85, 3, 1), (86, 3, 1), (256, 1, 1), (257, 2, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_around_the_number_of_rows_that_read_codes(n, h, hk, d):
    cache, g = _filled(3, 420, hk, d, 64, torch.float8_e4m3fn, seed=n)
    q = torch.randn(3, n, h, d, generator=g).bfloat16().to(DEV)
    for kw in ({}, dict(window=70, sink=9, cap=6.0)):
        lens = [420, n - 3, 131]
        _check_attention(W.attend_8bit(q, cache, _i32(lens), **kw), q, cache, lens, **kw)
        _check_attention(W.attend_8bit(q, cache, 300, **kw), q, cache, [300] * 3, **kw)


@pytest.mark.parametrize("n", [2, 80, 140])
def test_lengths_past_the_cache_under_a_window(n):
    """A length past the cache is the cache's, for what a long chunk reads back too: memory that is not written there holds NaN."""
    b, h, hk, d, cap = 3, 4, 2, 64, 500
    cache, g = _filled(b, cap, hk, d, 64, torch.int8, seed=41)
    q = torch.randn(b, n, h, d, generator=g).bfloat16().to(DEV)
    for kw in (dict(window=30), dict(window=30, sink=7)):
        for lens, x in (([cap + 40, 400, cap + 5000], None), ([cap + 100] * b, cap + 100)):
            waste = [torch.full((b, cap, hk, d), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(4)]
            del waste
            got = W.attend_8bit(q, cache, _i32(lens) if x is None else x, **kw)
            _check_attention(got, q, cache, [min(y, cap) for y in lens], **kw)


def test_ragged_lengths_that_move_between_replays():
    """Where a captured call's workgroups begin follows the lengths of each replay; two graphs in turn."""
    b, cap, hk, d = 4, 4000, 2, 128
    g = torch.Generator().manual_seed(51)
    sets = []
    for n, kw in ((1, {}), (3, dict(window=1200, sink=30))):
        cache, _ = _filled(b, cap, hk, d, 64, torch.int8, seed=n)
        q = torch.randn(b, n, 6, d, generator=g).bfloat16().to(DEV)
        lens = _i32([5, 0, 4000, 900])
        call = lambda cache=cache, q=q, lens=lens, kw=kw: W.attend_8bit(q, cache, lens, **kw)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        sets.append((graph, got, call, cache, q, lens, kw))
    for now in ([5, 0, 4000, 900], [0, 0, 0, 0], [4000, 4000, 4000, 4000], [1, 3999, 0, 64], [2000, 31, 33, 4005]):
        for graph, got, call, cache, q, lens, kw in sets:
            lens.copy_(_i32(now))
            graph.replay()
            torch.cuda.synchronize()
            want = call()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), now
            _check_attention(got, q, cache, [min(x, cap) for x in now], **kw)


def test_prompt_then_single_tokens():
    """A model's use of it all: a packed training step's attention, its prompt into the cache, drafts that are taken back, single tokens
    over all, some and the newest of the cache, against the same attention over the keys and values that the codes stand for."""
    b, h, hk, d, n = 2, 4, 2, 64, 300
    g = torch.Generator().manual_seed(20)
    make = lambda m, heads: torch.randn(b, m, heads, d, generator=g).bfloat16().to(DEV)  # noqa: E731
    q, k, v = make(n, h), make(n, hk), make(n, hk)
    slopes = torch.tensor([0.1, 0.05, 0.02, 0.01], device=DEV)
    lens = _i32([n, 211])
    cache = W.new_cache_8bit(b, 400, hk, d)
    W.kv_append_8bit(cache, k, v, 0, lengths=lens)
    held = W.kv_read_8bit(cache, 0, n)
    prompt = W.ranged_attention(q, *held, W.key_ranges(b, n, n, lengths=lens), cap=20.0, slopes=slopes)
    chunk, _ = W.attend_8bit(q[:, -140:], cache, n, cap=20.0, slopes=slopes)     # the same tokens, as the chunk of a longer prompt
    assert torch.equal(prompt[0, -140:], chunk[0])
    drafts = make(4, hk), make(4, hk)
    W.kv_append_8bit(cache, *drafts, lens)
    for step in range(3):
        new = make(1, hk), make(1, hk)
        W.kv_append_8bit(cache, *new, lens + step)
        at = (lens + step + 1).tolist()
        one = make(1, h)
        for kw in (dict(cap=20.0, slopes=slopes), dict(window=70, sink=4), dict(chosen=W.select_key_blocks(
                one, cache["k_block_sums"], lens + step + 1, block_size=64, topk=3))):
            _check_attention(W.attend_8bit(one, cache, lens + step + 1, **kw), one, cache, at, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,n", [(64, 3), (64, 40), (64, 300), (128, 16), (128, 150)])
def test_large_caps(dtype, d, n):
    """Scores far below the cap keep fp32's accuracy, also beside a query whose scores pass it, but for that of the one token that it sees: 0.
    Codes, and read back."""
    cache, g = _filled(1, n + 50, 1, d, 64, dtype, seed=n)
    cache["k"].view(torch.uint8)[:, 0, :, 0] = 0
    q = torch.randn(1, n, 2, d, generator=g).bfloat16().to(DEV)
    for cap in (100.0, 1100.0, 1e4, 1e6):
        far = q.clone()
        far[:, 0] = 0
        far[:, 0, :, 0] = 2 * cap * d ** 0.5
        for x, lens in ((q, n + 50), (far, n)):
            _check_attention(W.attend_8bit(x, cache, lens, cap=cap), x, cache, [lens], cap=cap)


def test_a_window_that_64_bits_barely_hold():
    """The library's own call: a window and a number of newest tokens whose sum passes 64 bits are as all tokens."""
    cache, _ = _filled(1, 130, 1, 64, 64, torch.int8, seed=60)
    _lib = W.cache8._lib
    c, _ = W.cache8._cache_args(cache)
    want = W.kv_read_8bit(cache, 0, 130)
    most = (1 << 63) - 1
    for last, window, sink in ((0, 0, 0), (most, most, 0), (most, 5, most), (3, most, most)):
        k, v = (torch.full((1, 130, 1, 64), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        _lib.launch("wa_kv8_read", _lib.Kv8ReadArgs(c, k.data_ptr(), v.data_ptr(), _lib.WA_BF16, 130, None, 0, None, 130, last, window, sink),
                    k.device)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1]), (last, window, sink)
    for start in (most, -most - 1, most - 100):      # all outside the cache: zeros
        _lib.launch("wa_kv8_read", _lib.Kv8ReadArgs(c, k.data_ptr(), v.data_ptr(), _lib.WA_BF16, 130, None, start, None, -1, 0, 0, 0), k.device)
        assert (k == 0).all() and (v == 0).all(), start


def test_a_chunk_over_a_cache_whose_offsets_pass_32_bits():
    """More rows than read codes: the far end is read back, and attended to at token offsets past 2^31."""
    cap, hk, d = (1 << 25) // 8 + 300, 8, 128
    n = W.cache8._FEW_ROWS + 4
    g = torch.Generator().manual_seed(16)
    cache = W.new_cache_8bit(1, cap, hk, d)
    k, v = (torch.randn(1, n, hk, d, generator=g).bfloat16().to(DEV) for _ in range(2))
    start = cap - n - 11
    W.kv_append_8bit(cache, k, v, start)
    first = start // 64 * 64
    small = W.new_cache_8bit(1, cap - first, hk, d)
    W.kv_append_8bit(small, k, v, start - first)
    q = torch.randn(1, n - 1, hk, d, generator=g).bfloat16().to(DEV)
    assert n - 1 > W.cache8._FEW_ROWS
    kw = dict(window=40, cap=6.0)     # the first query's window begins among the tokens that were never written, in both
    far = W.attend_8bit(q, cache, _i32([start + n]), **kw)
    _check_attention(W.attend_8bit(q, small, start - first + n, **kw), q, small, [start - first + n], **kw)
    lens = start - first + n
    want_k, want_v = W.kv_read_8bit(small, 0, small["k"].shape[1], dtype=torch.float32)
    want, want_lse = OC.attend(q[:, 64:], want_k, want_v, [lens], **kw)
    mag, _ = OC.attend(q[:, 64:], want_k, want_v.abs(), [lens], **kw)
    err = (far[0][:, 64:].cpu().double() - want).abs()
    assert (err <= U * mag + U * want.abs() + 2.0 ** -11 * mag).all()
    assert ((far[1][:, :, 64:].cpu().double() - want_lse).abs() <= 2.0 ** -12 + 2.0 ** -22 * want_lse.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,h", [(257, 1), (1, 257), (130, 2), (52, 5)])
def test_every_number_of_rows_that_are_read_back(dtype, d, n, h):
    """Chunks of just more rows than read codes, one token among them."""
    assert n * h > W.cache8._FEW_ROWS
    cache, g = _filled(1, 310, 1, d, 64, dtype, seed=n * h)
    q = torch.randn(1, n, h, d, generator=g).bfloat16().to(DEV)
    for kw in ({}, dict(window=40, sink=35, cap=4.0)):
        _check_attention(W.attend_8bit(q, cache, 301, **kw), q, cache, [301], **kw)
