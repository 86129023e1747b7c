"""``attend_selected`` on layouts of queries and caches that views make."""
import pytest
import torch

from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    cache = {name: torch.zeros(1, 300, 2, 64, dtype=torch.bfloat16, device=DEV) for name in "kv"}
    k, v = (torch.randn(1, 300, 2, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    W.kv_append(cache, k, v, write_start=0, block_size=64)
    return cache, torch.randn(1, n, 4, 64, generator=g).bfloat16().to(DEV)


def _same(cache, view, copy, **kw):
    got, want = (W.attend_selected(q, cache, 300, topk=3, **kw) for q in (view, copy))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].any()
    assert torch.equal(got[2].index, want[2].index) and torch.equal(got[2].num, want[2].num)


def test_queries_of_any_token_stride():
    """Queries are read at 64-bit offsets: neither one token's stride nor the distance between two is a reason to refuse."""
    cache, q = _case(1)
    far = torch.zeros(1 << 10, dtype=torch.bfloat16, device=DEV).as_strided((1, 1, 4, 64), (1 << 26, 1 << 25, 64, 1))
    far.copy_(q)
    _same(cache, far, q)
    cache, q = _case(2)
    apart = torch.zeros((1 << 25) + 512, dtype=torch.bfloat16, device=DEV).as_strided((1, 2, 4, 64), (1 << 26, 1 << 25, 64, 1))
    apart.copy_(q)
    _same(cache, apart, q)


@pytest.mark.parametrize("n", [1, 5, 70])
def test_queries_that_share_memory(n):
    """One query for all tokens and heads, and windows 8 elements apart."""
    cache, q = _case(n)
    one = q[:, :1, :1].expand(-1, n, 4, -1)
    _same(cache, one, one.contiguous())
    windows = q.flatten()[: 8 * (n * 4 - 1) + 64].as_strided((1, n, 4, 64), (0, 32, 8, 1))
    _same(cache, windows, windows.contiguous())


@pytest.mark.parametrize("n", [1, 5, 70])
def test_caches_whose_tokens_share_memory(n):
    """Keys and values of one row for all tokens, or overlapping: the bits of copies, the last block cut inside a tile."""
    cache, q = _case(n)
    for k in (cache["k"][:, :1].expand(-1, 300, -1, -1), cache["k"].flatten()[: 8 * 299 + 128].as_strided((1, 300, 2, 64), (0, 8, 64, 1))):
        sums = torch.zeros(1, 2, 5, 64, device=DEV)
        for j in range(5):
            sums[:, :, j] = k[:, 64 * j:64 * j + 64].float().sum(1)
        shared = {"k": k, "v": k, "k_block_sums": sums, "k_block_sums_block_size": 64}
        copies = {"k": k.clone(memory_format=torch.contiguous_format), "k_block_sums": sums, "k_block_sums_block_size": 64}
        copies["v"] = copies["k"]
        for kv_len in (300, 257, 33, n):
            got, want = (W.attend_selected(q, c, kv_len, topk=5) for c in (shared, copies))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,nb", [(1, 60), (1, 700), (1, 1500), (4, 60), (9, 700), (40, 700)])
def test_equal_key_sums_tie_in_every_launch(d, n, nb):
    """Blocks with one of five key sums: whole runs are chosen, and of the last one the lowest ids, for one query (either of
    its forms), a few and many."""
    g = torch.Generator().manual_seed(nb + n)
    kinds = torch.randn(2, 5, d, generator=g) * 30
    kind = torch.randint(0, 5, (2, nb), generator=g)
    sums = torch.stack([kinds[h, kind[h]] for h in range(2)])[None].to(DEV)
    q = torch.randn(1, n, 4, d, generator=g).bfloat16()
    got = W.select_key_blocks(q.to(DEV), sums, nb * 64, block_size=64, topk=nb // 3, sink_blocks=0, local_blocks=1)
    score = torch.einsum("nhd,hkd->nhk", q[0].double().view(n, 2, 2, d).sum(2), kinds.double())
    assert (score.sort(-1).values.diff(dim=-1) > 1e-6).all()      # five different scores, far beyond any rounding
    for i in range(n):
        last = (nb * 64 - n + i) // 64      # the query's own block
        for h in range(2):
            order = sorted(range(last), key=lambda j: (-score[i, h, kind[h, j]].item(), j))
            want = sorted(order[:nb // 3 - 1] + [last])
            assert got.index[0, i, h].tolist() == want and got.num[0, i, h].item() == nb // 3
