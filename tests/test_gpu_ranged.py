"""``key_ranges`` and ``ranged_attention`` against their 64-bit forms, forward and backward.

Ranges are whole numbers: equal. Attention, element by element, with u = 2^-8 (half a step of bf16): the weights are rounded once for
their product (u of M, the softmax-weighted |v|), the output once (u |y|), and scores are fp32 sums of D exact products, which
with the cap and the bias (magnitudes of at most 2^10 here) are off by less than 2^-12, so weights by 2^-11: u M + u |y| + 2^-11 M.
The log-sum-exp is of unrounded weights: 2^-12 + 2^-22 of its magnitude.

Gradients, with E_i = sum_d |o_i| |do_i|: delta is of the rounded output, off by u E_i (and D 2^-24 of it). dS is off by
P u E_i, by its own rounding u |dS| and the weight's as fp16, 2^-11 |dS|, and by the weight's error, 2^-11 P (|dP| + |delta|). The
gradients of q and k are sums of these times |k| and |q|, and are rounded once more; that of v is u + 2^-11 of the weighted |do|
and its rounding. The slopes' gradient comes from fp32 sums of unrounded terms: 2^-11 of P (|dP| + |delta|) |t - j|."""
import math

import pytest
import torch

from oracle import ranged as OR
from worldattention_amd import hsa as W

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8
TINY = 2.0 ** -100


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _ranges(b, n, m, rules):
    on_gpu = {k: _i32(v) if isinstance(v, list) else v for k, v in rules.items()}
    return W.key_ranges(b, n, m, device=DEV, **on_gpu)


def _mask_of(ranges, m):
    rows = ranges.rows
    assert ((rows[..., 0] <= rows[..., 1]) & (rows[..., 2] <= rows[..., 3])).all()
    return OR.of_runs(rows, m)


def _inputs(b, n, m, h, hk, d, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(*s, generator=g).mul(x).bfloat16().to(DEV) for s, x in (
        ((b, n, h, d), size), ((b, m, hk, d), size), ((b, m, hk, d), 1.0), ((b, n, h, d), 1.0)))
    return q, k, v, do


def check(q, k, v, do, ranges, mask, *, scale=None, cap=None, slopes=None, dlse=None, kv_len=None):
    """One call and its gradients against the definition."""
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)] + ([] if slopes is None else [slopes.detach().requires_grad_(True)])
    out, lse = W.ranged_attention(*leaves[:3], ranges, scale=scale, cap=cap, slopes=leaves[3] if slopes is not None else None, return_lse=True)
    outs, gouts = [out], [do]
    if dlse is not None:
        outs, gouts = [out, lse], [do, dlse]
    grads = torch.autograd.grad(outs, leaves, gouts)
    want64 = [t.detach().double().requires_grad_(True) for t in leaves]
    y, want_lse, (p, turn, far) = OR.attention(*want64[:3], mask, scale=scale, cap=cap, slopes=want64[3] if slopes is not None else None, kv_len=kv_len)
    fine = torch.isfinite(want_lse)
    loss = (y * do.double()).sum() + (0 if dlse is None else torch.where(fine, want_lse * dlse.double(), 0.0).sum())
    want = torch.autograd.grad(loss, want64)
    with torch.no_grad():
        h, hk = q.shape[2], k.shape[2]
        ka, va = (t.double().abs().transpose(1, 2).repeat_interleave(h // hk, 1) for t in (k, v))
        qa, doa = (t.double().abs().transpose(1, 2) for t in (q, do))
        big = torch.matmul(p, va).transpose(1, 2)
        err = (out.double() - y).abs()
        assert (err <= U * big + U * y.abs() + 2.0 ** -11 * big + TINY).all(), (err - U * big - U * y.abs()).max()
        assert torch.equal(torch.isinf(lse), ~fine)
        assert ((lse.double() - want_lse).abs()[fine] <= 2.0 ** -12 + 2.0 ** -22 * want_lse.abs()[fine]).all()
        assert (out.transpose(1, 2)[~fine] == 0).all() and (grads[0].transpose(1, 2)[~fine] == 0).all()
        s = q.shape[-1] ** -0.5 if scale is None else scale
        vh = v.double().transpose(1, 2).repeat_interleave(h // hk, 1)
        dp = torch.matmul(do.double().transpose(1, 2), vh.transpose(-1, -2).contiguous())
        delta = (p * dp).sum(-1, keepdim=True)
        shift = 0.0 if dlse is None else torch.where(fine, dlse.double(), 0.0)[..., None]
        e = (y.abs() * do.double().abs()).sum(-1).transpose(1, 2)[..., None]
        ds = p * (dp - delta + shift)
        wide = p * (dp.abs() + delta.abs() + abs(shift))
        off = ((U + 2.0 ** -10) * ds.abs() + p * U * e + 2.0 ** -11 * wide) * (turn + 2.0 ** -20) * s
        group = lambda x: x.view(x.shape[0], hk, h // hk, *x.shape[2:]).sum(2).transpose(1, 2)  # noqa: E731
        bounds = [torch.matmul(off, ka).transpose(1, 2), group(torch.matmul(off.transpose(-1, -2).contiguous(), qa)),
                  group(torch.matmul(p.transpose(-1, -2).contiguous(), doa)) * (U + 2.0 ** -11)]
        if slopes is not None:
            bounds.append((2.0 ** -11 * wide * far).sum((0, 2, 3)))
        for name, got, w, bound in zip(("dq", "dk", "dv", "dslopes"), grads, want, bounds):
            last = U if name != "dslopes" else 2.0 ** -22
            err = (got.double() - w).abs()
            assert (err <= bound + last * w.abs() + TINY).all(), (name, (err - bound - last * w.abs()).max())
    return out, lse, grads


RULES = [dict(), dict(causal=False), dict(chunk=7), dict(window=5), dict(window=70, sink=3), dict(causal=False, window=9),
         dict(prefix=10), dict(window=3, sink=2, prefix=4), dict(causal=False, window=4, prefix=6, sink=5), dict(chunk=50, window=20, sink=1)]


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("b,n,m", [(1, 1, 1), (2, 65, 65), (3, 64, 130), (1, 130, 70), (2, 1, 200)])
def test_ranges_hold_what_the_rules_say(rules, b, n, m):
    for more in (dict(), dict(documents=[0, 17, 17, 60, 64]), dict(documents=[[3, 30, 50], [0, 64, 65], [5, 5, 200]][:b]),
                 dict(lengths=[m, 0, m // 2][:b]), dict(kv_len=[m, m // 3, -4][:b]), dict(prefix=[0, 9, 500][:b]), dict(kv_len=m - 1)):
        both = {**rules, **more}
        got = _ranges(b, n, m, both)
        assert torch.equal(_mask_of(got, m).expand(b, n, m), OR.seen(b, n, m, **both)), both
        _check_tiles(got, n, m)


def _check_tiles(ranges, n, m):
    """The summaries hold every row's runs, and name as held by all rows only what all hold."""
    rows, tiles = ranges.rows.cpu().long(), ranges.tiles.cpu().long()
    for b in range(rows.shape[0]):
        for i in range(tiles.shape[1]):
            r, t = rows[b, 64 * i: 64 * i + 64], tiles[b, i].tolist()
            for run in range(2):
                has = r[:, 2 * run + 1] > r[:, 2 * run]
                lo = int(r[has, 2 * run].min()) if has.any() else 0
                hi = int(r[has, 2 * run + 1].max()) if has.any() else 0
                assert (t[2 * run], t[2 * run + 1]) == (lo, hi)
                if has.all():
                    assert (t[4 + 2 * run], t[5 + 2 * run]) == (int(r[:, 2 * run].max()), int(r[:, 2 * run + 1].min()))
                else:
                    assert t[4 + 2 * run] > t[5 + 2 * run]
            some = ((r[:, 1] > r[:, 0]) | (r[:, 3] > r[:, 2])).nonzero()
            assert t[8] == (64 * i + int(some.max()) + 1 if len(some) else 0)


def test_given_runs_are_put_in_order():
    g = torch.Generator().manual_seed(3)
    given = torch.randint(-20, 320, (2, 150, 4), generator=g, dtype=torch.int32)
    given[0, :20] = 0
    given[1, 5] = torch.tensor([2 ** 31 - 1, -2 ** 31, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)
    got = W.key_ranges(2, 150, 300, given=given.to(DEV))
    assert torch.equal(_mask_of(got, 300), OR.of_runs(given, 300))
    rows = got.rows.cpu()
    both = (rows[..., 3] > rows[..., 2]) & (rows[..., 1] > rows[..., 0])
    assert both.any() and (rows[..., 3] < rows[..., 0])[both].all()
    _check_tiles(got, 150, 300)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,n,m,h,hk,rules", [
    (1, 1, 1, 1, 1, dict()), (2, 3, 3, 4, 2, dict()), (1, 64, 64, 2, 1, dict()), (1, 129, 129, 3, 3, dict()),
    (2, 333, 333, 4, 2, dict(prefix=100)), (1, 200, 517, 2, 2, dict(causal=False)), (1, 517, 200, 2, 1, dict()),
    (2, 300, 300, 4, 1, dict(documents=[0, 40, 41, 170, 290])), (2, 257, 257, 2, 2, dict(lengths=[257, 131])),
    (1, 400, 400, 2, 2, dict(window=70, sink=5)), (1, 390, 390, 2, 1, dict(chunk=130)), (2, 100, 700, 2, 2, dict(window=300, sink=64, kv_len=[650, 90])),
    (1, 256, 256, 1, 1, dict(window=1)), (1, 320, 320, 2, 2, dict(causal=False, window=33, prefix=20))])
def test_forward_and_gradients(d, b, n, m, h, hk, rules):
    q, k, v, do = _inputs(b, n, m, h, hk, d, seed=n + m)
    ranges = _ranges(b, n, m, rules)
    check(q, k, v, do, ranges, OR.seen(b, n, m, **rules))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap,slopes,dlse", [(30.0, False, False), (None, True, False), (5.0, True, True), (None, False, True), (0.5, True, False)])
def test_caps_slopes_and_the_log_sum_exps_gradient(d, cap, slopes, dlse):
    b, n, m, h, hk = 2, 210, 330, 4, 2
    q, k, v, do = _inputs(b, n, m, h, hk, d, seed=5, size=2.0)
    rules = dict(window=150, sink=7, kv_len=[330, 201])
    ranges = _ranges(b, n, m, rules)
    g = torch.Generator().manual_seed(1)
    check(q, k, v, do, ranges, OR.seen(b, n, m, **rules), cap=cap, scale=0.11, kv_len=rules["kv_len"],
          slopes=torch.tensor([0.5, 0.0, 0.03, -0.01], device=DEV) if slopes else None,
          dlse=torch.randn(b, h, n, generator=g).to(DEV) if dlse else None)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("part", [0.1, 0.29, 0.31, 0.49, 0.51, 1.5])
def test_scores_at_parts_of_the_cap(d, part):
    """The largest score at some part of the cap, on either side of where a tile's scores take another form of the tanh."""
    b, n, h, hk = 1, 200, 2, 1
    q, k, v, do = _inputs(b, n, n, h, hk, d, seed=44, size=1.5)
    most = (torch.matmul(q.double().transpose(1, 2), k.double().transpose(1, 2).transpose(2, 3).contiguous()) * 0.2).abs().max().item()
    check(q, k, v, do, _ranges(b, n, n, dict()), OR.seen(b, n, n), cap=most / part, scale=0.2)


def test_given_runs_in_attention():
    """Any runs: rows that see nothing between rows that see much, runs that overlap, two far apart."""
    g = torch.Generator().manual_seed(9)
    b, n, m = 2, 200, 450
    given = torch.randint(-40, 500, (b, n, 4), generator=g, dtype=torch.int32)
    given[0, 30:110] = 0
    given[1, :, 2:] = torch.tensor([10, 20], dtype=torch.int32)
    given[1, :, :2] = torch.tensor([400, 430], dtype=torch.int32)
    q, k, v, do = _inputs(b, n, m, 2, 1, 128, seed=2)
    check(q, k, v, do, W.key_ranges(b, n, m, given=given.to(DEV)), OR.of_runs(given, m), slopes=torch.tensor([0.01, 0.1], device=DEV))
    shared = W.key_ranges(b, n, m, given=given[:1].to(DEV))
    check(q, k, v, do, shared, OR.of_runs(given[:1], m))


@pytest.mark.parametrize("d", [16, 80, 100])
def test_padded_head_dims(d):
    q, k, v, do = _inputs(1, 150, 150, 2, 1, d, seed=d)
    check(q, k, v, do, _ranges(1, 150, 150, dict()), OR.seen(1, 150, 150), cap=20.0)


def test_a_single_key_leaves_no_gradient_of_scores():
    """A row's only key has weight 1 whatever its score: zeros, not roundings."""
    q, k, v, do = _inputs(1, 300, 300, 2, 1, 128, seed=4)
    for rules in (dict(window=1), dict(documents=list(range(301)))):
        _, _, grads = check(q, k, v, do, _ranges(1, 300, 300, rules), OR.seen(1, 300, 300, **rules), slopes=torch.full((2,), 0.1, device=DEV))
        assert all((x == 0).all() for x in (grads[0], grads[1], grads[3]))


def test_any_strides():
    """Heads outside tokens, a slice of a fused projection, a key head shared by expansion, gradients of any stride."""
    b, n, h, d = 2, 140, 4, 64
    g = torch.Generator().manual_seed(7)
    fused = torch.randn(b, n, 3 * h * d + 8, generator=g).bfloat16().to(DEV)
    q, k, v = (fused[..., i * h * d + 8: (i + 1) * h * d + 8].view(b, n, h, d) for i in range(3))
    do = torch.randn(b, h, n, d, generator=g).bfloat16().to(DEV).transpose(1, 2)
    ranges, mask = _ranges(b, n, n, dict(prefix=9)), OR.seen(b, n, n, prefix=9)
    check(q, k, v, do, ranges, mask)
    check(q, k[:, :, :1].expand(b, n, h, d), v[:, :, 1:2].expand(b, n, h, d), do, ranges, mask)
    odd = torch.randn(b, n, h, d + 1, generator=g).bfloat16().to(DEV)[..., 1:]   # rows on odd addresses
    check(odd, k, v, odd, ranges, mask)
    first = q[:1].expand(b, n, h, d)
    check(first, k, v, do, ranges, mask)


def test_padding_is_not_read():
    """NaN and infinities behind every sequence leave results and gradients as they are."""
    b, n, h, d = 2, 300, 2, 128
    q, k, v, do = _inputs(b, n, n, h, 1, d, seed=11)
    lengths = [211, 64]
    ranges = _ranges(b, n, n, dict(lengths=lengths))
    clean = check(q, k, v, do, ranges, OR.seen(b, n, n, lengths=lengths))
    for i, x in enumerate(lengths):
        for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan), (do, math.nan)):
            t[i, x:] = bad
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out, lse = W.ranged_attention(*leaves, ranges, return_lse=True)
    grads = torch.autograd.grad(out, leaves, do)
    for got, want in zip((out, lse, *grads), (clean[0], clean[1], *clean[2])):
        assert torch.equal(got, want)


def test_many_row_tiles_are_listed_in_parts():
    """More than 65,536 rows; a stretch of them against the definition."""
    n, d, w, a = 66200, 64, 90, 65200
    g = torch.Generator().manual_seed(13)
    q, k, v, do = (torch.randn(1, n, 1, d, generator=g).bfloat16().to(DEV) for _ in range(4))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = W.ranged_attention(*leaves, _ranges(1, n, n, dict(window=w)))
    grads = torch.autograd.grad(out, leaves, do)
    part = [t.detach()[:, a:] for t in (q, k, v)]
    mask = OR.seen(1, n - a, n - a, window=w)
    some, _, some_grads = check(*part, do[:, a:], _ranges(1, n - a, n - a, dict(window=w)), mask)
    assert torch.allclose(out[:, a + w:].float(), some[:, w:].float(), atol=2.0 ** -6)
    for got, want in zip(grads, some_grads):
        assert torch.allclose(got[:, a + 2 * w:].float(), want[:, 2 * w:].float(), rtol=2.0 ** -5, atol=2.0 ** -5)


def test_gradients_against_differences():
    """The directional derivative of the 64-bit loss, by central differences, along the gradient itself."""
    b, n, h, d = 1, 90, 2, 64
    q, k, v, do = _inputs(b, n, n, h, 1, d, seed=17)
    ranges, mask = _ranges(b, n, n, dict(window=40, sink=3)), OR.seen(b, n, n, window=40, sink=3)
    slopes = torch.tensor([0.2, 0.05], device=DEV)
    _, _, grads = check(q, k, v, do, ranges, mask, cap=4.0, slopes=slopes)
    x = [t.double() for t in (q, k, v, slopes)]
    loss = lambda y: (OR.attention(*y[:3], mask, cap=4.0, slopes=y[3])[0] * do.double()).sum()  # noqa: E731
    for i, g in enumerate(grads):
        step = 1e-5 * g.double() / g.double().norm()
        up, down = ([t + s * step if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        slope = float(loss(up) - loss(down)) / 2e-5
        # along the gradient the derivative is its norm: off by what its rounded elements are off, at most 2^-6 of it here
        assert abs(slope - float(g.double().norm())) <= 2.0 ** -6 * abs(slope), (i, slope, float(g.double().norm()))


def test_calls_without_tokens():
    q, k, v, _ = _inputs(2, 5, 7, 2, 1, 64)
    e = lambda t: t[:, :0].detach().requires_grad_(True)  # noqa: E731
    out, lse = W.ranged_attention(q.requires_grad_(True), e(k), e(v), _ranges(2, 5, 0, dict()), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert (torch.autograd.grad(out.sum(), q)[0] == 0).all()
    qe, kg = e(q), k.detach().requires_grad_(True)
    out = W.ranged_attention(qe, kg, v, _ranges(2, 0, 7, dict()))
    assert out.shape == (2, 0, 2, 64)
    assert (torch.autograd.grad(out.sum(), kg)[0] == 0).all()
    assert W.ranged_attention(q[:0].detach(), k[:0].detach(), v[:0], _ranges(0, 5, 7, dict())).shape == (0, 5, 2, 64)


def test_repeats_give_the_same_bits_and_other_streams_too():
    b, n, h, d = 2, 500, 4, 128
    q, k, v, do = _inputs(b, n, n, h, 2, d, seed=21)
    slopes = torch.rand(h, device=DEV)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, slopes)]
        out, lse = W.ranged_attention(*leaves[:3], _ranges(b, n, n, dict(window=200, sink=4)), cap=9.0, slopes=leaves[3], return_lse=True)
        return out, lse, *torch.autograd.grad(out, leaves, do)

    first, side = once(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    for x, y, z in zip(first, other, once()):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_captured_steps():
    """Two captured training steps with ranges of device lengths, replayed in turn with changed inputs between eager work."""
    b, n, h, d = 2, 200, 2, 64
    sets = []
    for seed in (1, 2):
        q, k, v, do = _inputs(b, n, n, h, 1, d, seed=seed)
        lengths = _i32([200, 50 * seed])

        def step(q=q, k=k, v=v, do=do, lengths=lengths):
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
            out = W.ranged_attention(*leaves, W.key_ranges(b, n, n, lengths=lengths), cap=7.0)
            return out.detach(), *torch.autograd.grad(out, leaves, do)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        sets.append((graph, got, step, (q, k, v, do, lengths)))
    for turn in range(3):
        for graph, got, step, data in sets:
            data[0].mul_(1.1)
            data[4][0] = 60 + 40 * turn
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(got, step()):
                assert torch.equal(x, y), turn


def test_ranges_keep_what_they_were_made_from():
    """Lengths that a program counts up after the ranges were made change neither the rows nor their positions."""
    b, n = 2, 100
    q, k, v, _ = _inputs(b, n, n, 2, 2, 64, seed=30)
    lens, slopes = _i32([100, 60]), torch.tensor([0.3, 0.1], device=DEV)
    ranges = W.key_ranges(b, n, n, kv_len=lens)
    first = W.ranged_attention(q, k, v, ranges, slopes=slopes)
    lens += 7
    assert torch.equal(first, W.ranged_attention(q, k, v, ranges, slopes=slopes))


@pytest.mark.parametrize("dlse", [False, True])
def test_single_keys_with_the_log_sum_exps_gradient(dlse):
    """One key: the weight's gradient is 0, the log-sum-exp's is its score's."""
    q, k, v, do = _inputs(1, 200, 200, 2, 2, 64, seed=31)
    g = torch.Generator().manual_seed(2)
    check(q, k, v, do, _ranges(1, 200, 200, dict(window=1)), OR.seen(1, 200, 200, window=1), cap=6.0,
          slopes=torch.tensor([0.2, 0.1], device=DEV), dlse=torch.randn(1, 2, 200, generator=g).to(DEV) if dlse else None)


@pytest.mark.parametrize("n,m", [(5, 4000), (130, 5000)])
def test_few_rows_over_many_keys(n, m):
    """Launches whose rows are too few to fill the GPU: steps in parts, joined; keys in runs."""
    q, k, v, do = _inputs(1, n, m, 2, 1, 128, seed=n)
    for rules in (dict(), dict(window=700, sink=40), dict(kv_len=[m - 64])):
        check(q, k, v, do, _ranges(1, n, m, rules), OR.seen(1, n, m, **rules), cap=15.0)


def test_offsets_that_pass_32_bits():
    """Sequences and heads further apart than 2^31 elements."""
    n, d = 150, 64
    g = torch.Generator().manual_seed(33)
    pool = torch.zeros(((1 << 31) + 4096 * 64,), dtype=torch.bfloat16, device=DEV)
    far = torch.as_strided(pool, (2, n, 1, d), ((1 << 31) + 64, 2 * d, d, 1))
    far.copy_(torch.randn(2, n, 1, d, generator=g))
    q, k, v, do = _inputs(2, n, n, 1, 1, d, seed=34)
    check(far, far, far, do, _ranges(2, n, n, dict()), OR.seen(2, n, n))


def test_scores_at_the_ends_of_fp32():
    """Scores near the lowest numbers of fp32 still weigh their keys; infinite ones give NaN, as a softmax of them does."""
    n, d = 70, 64
    q, k, v, _ = _inputs(1, n, n, 1, 1, d, seed=35)
    q.fill_(1.0)
    k.zero_()
    k[..., 0] = -3.0e38
    out, lse = W.ranged_attention(q, k, v, _ranges(1, n, n, dict()), scale=0.5, return_lse=True)
    want = torch.cumsum(v[0, :, 0].double(), 0) / torch.arange(1, n + 1, device=DEV)[:, None]
    assert ((out[0, :, 0].double() - want).abs() <= 2.0 ** -7 * (1 + want.abs())).all() and lse.isfinite().all()
    k[0, 40, 0, 1] = math.inf
    out = W.ranged_attention(q, k, v, _ranges(1, n, n, dict(documents=[0, 40, 41, 70])))
    assert out[0, 40].isnan().all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap", [100.0, 1024.0, 1100.0, 3e3, 1e4, 1e5, 1e6])
@pytest.mark.parametrize("far", [False, True])
def test_large_caps(d, cap, far):
    """Scores far below the cap keep fp32's accuracy, also beside a row whose scores pass it, but for that of the one key that it sees: 0."""
    b, n, h, hk = 1, 200, 2, 1
    q, k, v, do = _inputs(b, n, n, h, hk, d, seed=52)
    if far:
        q[:, 0] = 0
        q[:, 0, :, 0] = 2 * cap * d ** 0.5
        k[:, 0, :, 0] = 0
    check(q, k, v, do, _ranges(b, n, n, dict()), OR.seen(b, n, n), cap=cap, slopes=torch.tensor([0.1, 0.01], device=DEV))


@pytest.mark.parametrize("power,cap", [(-100, 5.0), (-60, 1e4), (-13, 1000.0), (-16, 1000.0), (40, 3.0), (80, 1e-6), (18, 10.0), (19, 10.0), (21, 10.0), (28, 900.0), (-4, 10.0), (-9, 10.0)])
def test_caps_at_any_scale(power, cap):
    """Scores of about 1 from small and large products."""
    b, n, h, hk, d = 1, 130, 2, 1, 64
    q, k, v, do = _inputs(b, n, n, h, hk, d, seed=53, size=2.0 ** -(power // 2))
    check(q, k, v, do, _ranges(b, n, n, dict()), OR.seen(b, n, n), scale=2.0 ** (power - 3), cap=cap)


@pytest.mark.parametrize("rules", RULES)
def test_documents_that_begin_before_the_first_token(rules):
    """Chunks, sinks and prefixes count from the document's border, tokens that are no longer held among them."""
    for documents in ([-5, 40, 70], [-200, -7, 30, 65], [[-3, 66, 70], [0, 9, 70]]):
        both = {**rules, "documents": documents}
        got = _ranges(2, 70, 70, both)
        assert torch.equal(_mask_of(got, 70).expand(2, 70, 70), OR.seen(2, 70, 70, **both)), both
        _check_tiles(got, 70, 70)
