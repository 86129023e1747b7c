"""Attention under masks, caps and distance biases, and the 8-bit cache that serves it.

They carry a causal model that trains on packed or chunked sequences and then decodes from a cache of
half the size: every layer's training step and prompt runs ``ranged`` attention (each row sees up to two
runs of keys: its document, its frame, its window, the sinks or the prefix); its new keys and values go
into a ``cache`` of 8-bit codes with a scale for each block of tokens and head, and are ``read`` back from
it; and its newest tokens ``attend`` to that cache. Each case is one call of such a layer.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # A small model on short sequences with a seen prefix and learnt distance slopes: launches and host time decide it.
        _ranged("ranged_train_small", "train", 2, 333, 333, 4, 2, 64, prefix=100, slopes="learnt"),
        # Training on one chunk of a video, 3 frames of 30 x 52 latent tokens: a token sees its frame and those before it.
        _ranged("ranged_train_frames", "train", 1, 4680, 4680, 12, 12, 128, chunk=1560),
        # Packed documents with a padded end, capped scores and slopes, shared key heads.
        _ranged("ranged_train_packed", "train", 1, 8190, 8190, 16, 4, 128, docs=7, score_cap=30.0, slopes="fixed"),
        # The whole window of 21 frames as one causal prompt.
        _ranged("ranged_prompt_window", "forward", 1, 32760, 32760, 12, 12, 128),
        # One token of each of 64 sequences written behind ragged lengths, and its block read back: latency.
        _cache("cache_step", 64, 1, 8, 128, 64, "int8", 1024, True),
        # A padded batch of prompts written, and read back as written.
        _cache("cache_prompt", 4, 4680, 12, 128, 128, "e4m3", 4992, True),
        # One block of one sequence handed to another path.
        _read("read_block", 1, 64, 8, 128, 64, "e4m3", 1024, "float32"),
        # A whole window of a layer handed to a path that reads bf16.
        _read("read_window", 1, 32760, 12, 128, 64, "int8", 32768, "bfloat16"),
        # One token of one sequence over a short cache: latency.
        _attend("attend_step", 1, 1, 32, 8, 128, 64, "int8", 4096),
        # One token each of a served batch of ragged sequences: the cache is read once.
        _attend("attend_batch", 32, 1, 32, 8, 128, 64, "int8", 32768, ragged=True),
        # Four drafted tokens of each of 8 ragged sequences that attend to their chosen blocks.
        _attend("attend_chosen", 8, 4, 32, 8, 128, 64, "e4m3", 32768, ragged=True, topk=32),
        # A chunk of a long prompt with a window, sinks, capped scores and slopes.
        _attend("attend_prompt", 1, 1024, 32, 8, 128, 64, "int8", 16384, window=8192, sink=64, score_cap=50.0, slopes=True),
    ]


def _ranged(name, direction, batch, queries, length, heads, kv_heads, dim, causal=True, chunk=1, window=0, sink=0, prefix=0,
            docs=0, score_cap=0.0, slopes="none"):
    return _named(name, dict(kind="ranged", direction=direction, batch=batch, queries=queries, length=length, heads=heads,
                             kv_heads=kv_heads, dim=dim, causal=causal, chunk=chunk, window=window, sink=sink, prefix=prefix,
                             docs=docs, score_cap=score_cap, slopes=slopes))


def _cache(name, batch, tokens, kv_heads, dim, block, codes, cap, ragged):
    return _named(name, dict(kind="cache", batch=batch, tokens=tokens, kv_heads=kv_heads, dim=dim, block=block, codes=codes,
                             cap=cap, ragged=ragged))


def _read(name, batch, tokens, kv_heads, dim, block, codes, cap, out):
    return _named(name, dict(kind="read", batch=batch, tokens=tokens, kv_heads=kv_heads, dim=dim, block=block, codes=codes,
                             cap=cap, out=out))


def _attend(name, batch, queries, heads, kv_heads, dim, block, codes, cap, ragged=False, topk=0, window=0, sink=0,
            score_cap=0.0, slopes=False):
    return _named(name, dict(kind="attend", batch=batch, queries=queries, heads=heads, kv_heads=kv_heads, dim=dim, block=block,
                             codes=codes, cap=cap, ragged=ragged, topk=topk, window=window, sink=sink, score_cap=score_cap,
                             slopes=slopes))


def _named(name, case):
    return case if name is None else dict(name=name, **case)


def _spread(rng, low, high):
    """A whole number, even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["ranged", "ranged", "ranged", "cache", "read", "attend", "attend", "attend"])
    codes, block, dim = rng.choice(["int8", "e4m3"]), rng.choice([64, 128]), rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    if kind == "ranged":
        direction = rng.choice(["forward", "train", "train"])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        batch = rng.randint(1, 3)
        # as many pairs of tokens and heads as the largest listed case of the direction has
        pairs = 12 * 32760 ** 2 // 2 if direction == "forward" else 16 * 8190 ** 2 // 7
        length = _spread(rng, 1, min(32760, math.isqrt(pairs // (heads * batch))))
        queries = length if rng.random() < 0.7 else rng.randint(1, length)
        causal = rng.random() < 0.8
        return _ranged(None, direction, batch, queries, length, heads, kv_heads, rng.choice([64, 80, 128, 128]), causal,
                       rng.choice([1, 1, 1, rng.randint(2, 1560)]) if causal else 1,
                       rng.choice([0, 0, _spread(rng, 1, length)]), rng.choice([0, 0, rng.randint(1, 70)]),
                       rng.choice([0, 0, rng.randint(1, length)]), rng.choice([0, 0, rng.randint(1, 9)]),
                       rng.choice([0.0, 0.0, 30.0, 50.0]), rng.choice(["none", "none", "fixed", "learnt"]))
    if kind == "cache":
        batch = _spread(rng, 1, 64)
        tokens = 1 if rng.random() < 0.4 else _spread(rng, 2, max(2, 224640 // (batch * kv_heads)))
        return _cache(None, batch, tokens, kv_heads, dim, block, codes, tokens + rng.randint(0, 400), rng.random() < 0.7)
    if kind == "read":
        batch = rng.randint(1, 8)
        tokens = _spread(rng, 1, min(32768, 393120 // (batch * kv_heads)))
        return _read(None, batch, tokens, kv_heads, dim, block, codes, tokens + rng.randint(0, 300),
                     rng.choice(["bfloat16", "float32"]))
    batch, queries = (_spread(rng, 1, 32), rng.randint(1, 8)) if rng.random() < 0.7 else (1, _spread(rng, 9, 1024))
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    cap = _spread(rng, 1, min(131072, 8 * 1048576 // (batch * kv_heads), 16384 * 32 * 1024 // (queries * heads)))
    topk = rng.choice([0, 0, rng.randint(1, 32)]) if queries <= 8 else 0
    window, sink = (0, 0) if topk or rng.random() < 0.5 else (_spread(rng, 1, cap), rng.randint(0, 130))
    return _attend(None, batch, min(queries, cap), heads, kv_heads, dim, block, codes, cap, batch > 1, topk, window, sink,
                   rng.choice([0.0, 0.0, 30.0, 50.0]), rng.random() < 0.3)


def _documents(case):
    """Document borders in a sequence of ``length`` tokens: uneven documents that leave its last 3% as padding."""
    if not case["docs"]:
        return None
    r = random.Random(case["docs"] * 1000003 + case["length"])
    parts = [r.uniform(0.2, 2.0) for _ in range(case["docs"])]
    end = case["length"] - case["length"] // 32
    at = np.concatenate(([0.0], np.cumsum(parts))) / sum(parts)
    return [int(x) for x in np.floor(at * end + 1e-6)]


def _kv_lengths(case):
    """A served batch's lengths: the whole cache, or spread from it down to less than the new tokens."""
    b, cap = case["batch"], case["cap"]
    return [max(0, cap - (cap * i) // (b - 1)) if case["ragged"] and b > 1 else cap for i in range(b)]


def _written(case):
    """Where a batch's new tokens go, and how many each sequence brings (one brings none in a padded batch)."""
    b, n, room = case["batch"], case["tokens"], case["cap"] - case["tokens"]
    starts = [room * (i + 1) // b if case["ragged"] else room for i in range(b)]
    counts = [n - (n * i) // (b - 1) if case["ragged"] and b > 1 and n > 1 else n for i in range(b)]
    return starts, counts


# ------------------------------------------------------------------------------------------------
# What a program has in hand before the call
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"ranged": _prepare_ranged, "cache": _prepare_cache, "read": _prepare_read, "attend": _prepare_attend}[
        case["kind"]](case, g)


def _normal(g, shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _slopes(heads):
    """Slopes from 1/2 down to 1/256 over the heads."""
    return torch.exp2(-1.0 - 7.0 * torch.arange(heads, device=DEV, dtype=torch.float32) / max(1, heads - 1))


def _prepare_ranged(case, g):
    b, n, m, h, hk, d = (case[x] for x in ("batch", "queries", "length", "heads", "kv_heads", "dim"))
    train = case["direction"] == "train"
    s = dict(case=case, train=train, q=_normal(g, (b, n, h, d)), k=_normal(g, (b, m, hk, d)), v=_normal(g, (b, m, hk, d)),
             slopes=None if case["slopes"] == "none" else _slopes(h), documents=None)
    docs = _documents(case)
    if docs:
        s["documents"] = torch.tensor(docs, dtype=torch.int32, device=DEV)
    if case["slopes"] == "learnt":
        s["slopes"] *= 1 + 0.1 * torch.rand((h,), generator=g, device=DEV)
    if train:
        s["dout"] = _normal(g, (b, n, h, d))
    if own:
        from worldattention_amd.hsa import key_ranges

        # made once for a batch and used by every layer
        s["ranges"] = key_ranges(b, n, m, causal=case["causal"], chunk=case["chunk"], window=case["window"] or None,
                                 sink=case["sink"], prefix=case["prefix"], documents=s["documents"], device=DEV)
        if train:
            for name in ("q", "k", "v"):
                s[name].requires_grad_(True)
            if case["slopes"] == "learnt":
                s["slopes"].requires_grad_(True)
    return s


def _tokens(case, g, tokens):
    """Keys or values whose channels differ in size, as a trained layer's do."""
    size = torch.exp2(1.5 * torch.randn((case["kv_heads"], case["dim"]), generator=g, device=DEV))
    return (torch.randn((case["batch"], tokens, case["kv_heads"], case["dim"]), generator=g, device=DEV) * size).bfloat16()


def _empty_cache(case):
    b, cap, hk, d, bs = (case[x] for x in ("batch", "cap", "kv_heads", "dim", "block"))
    nb = -(-cap // bs)
    codes = dict(dtype=torch.uint8, device=DEV)
    return {"k": torch.zeros((b, cap, hk, d), **codes).view(CODES[case["codes"]]),
            "v": torch.zeros((b, cap, hk, d), **codes).view(CODES[case["codes"]]),
            "k_scale": torch.zeros((b, hk, nb), device=DEV), "v_scale": torch.zeros((b, hk, nb), device=DEV),
            "k_block_sums": torch.zeros((b, hk, nb, d), device=DEV), "k_block_sums_block_size": bs}


def _filled_cache(case, g):
    """A cache whose blocks were each written whole."""
    c = _empty_cache(case)
    b, cap, hk, d, bs = (case[x] for x in ("batch", "cap", "kv_heads", "dim", "block"))
    nb = -(-cap // bs)
    size = {x: torch.exp2(0.5 * torch.randn((hk, d), generator=g, device=DEV)) for x in "kv"}
    for i in range(b):
        for x in "kv":
            t = torch.randn((cap, hk, d), generator=g, device=DEV).mul_(size[x])
            t = torch.nn.functional.pad(t, (0, 0, 0, 0, 0, nb * bs - cap)).view(nb, bs, hk, d)
            scale = _needed_scale(t.abs().amax((1, 3)), LARGEST[case["codes"]])          # [nb, Hk]
            codes = _encode(t / scale[:, None, :, None], case["codes"])
            c[x].view(torch.uint8)[i] = codes.view(torch.uint8).view(nb * bs, hk, d)[:cap]
            c[x + "_scale"][i] = scale.T
            if x == "k":
                c["k_block_sums"][i] = (codes.float().sum(1) * scale[..., None]).transpose(0, 1)
    return c


def _prepare_cache(case, g):
    starts, counts = _written(case)
    c, bs = _empty_cache(case), case["block"]
    s = dict(case=case, cache=c, start=torch.tensor(starts, dtype=torch.int32, device=DEV),
             counts=torch.tensor(counts, dtype=torch.int32, device=DEV) if case["ragged"] else None,
             k=_tokens(case, g, case["tokens"]), v=_tokens(case, g, case["tokens"]))
    s["first"] = s["start"] // bs * bs      # the first written block's first token
    before = {x: _tokens(case, g, bs) for x in "kv"}
    for i, start in enumerate(starts):      # that block's earlier tokens, in codes and scales of their own
        n = start % bs
        if not n:
            continue
        for x in "kv":
            t = before[x][i, :n].float()
            scale = _needed_scale(t.abs().amax((0, 2)), LARGEST[case["codes"]])
            codes = _encode(t / scale[:, None], case["codes"])
            c[x].view(torch.uint8)[i, start - n: start] = codes.view(torch.uint8)
            c[x + "_scale"][i, :, start // bs] = scale
            if x == "k":
                c["k_block_sums"][i, :, start // bs] = codes.float().sum(0) * scale[:, None]
    return s


def _prepare_read(case, g):
    starts = [(case["cap"] - case["tokens"]) * (i + 1) // case["batch"] for i in range(case["batch"])]
    return dict(case=case, cache=_filled_cache(case, g), start=torch.tensor(starts, dtype=torch.int32, device=DEV))


def _prepare_attend(case, g):
    b, n, h, hk, d, cap, bs = (case[x] for x in ("batch", "queries", "heads", "kv_heads", "dim", "cap", "block"))
    s = dict(case=case, q=_normal(g, (b, n, h, d)), cache=_filled_cache(case, g), slopes=_slopes(h) if case["slopes"] else None,
             lengths=torch.tensor(_kv_lengths(case), dtype=torch.int32, device=DEV), index=None, num=None)
    if case["topk"]:
        # a choice in ascending order: each query's last block, and others drawn from those before it
        nb, topk = -(-cap // bs), case["topk"]
        seen = (s["lengths"][:, None] - n + 1 + torch.arange(n, device=DEV)).clamp(min=0)
        blocks = ((seen + bs - 1) // bs)[:, :, None, None]
        j = torch.arange(nb, device=DEV)
        rank = torch.rand((b, n, hk, nb), generator=g, device=DEV)
        rank = torch.where(j == blocks - 1, 2.0, torch.where(j < blocks, rank, -1.0))
        pick = rank.sort(-1, descending=True).indices[..., :topk]
        pick = torch.nn.functional.pad(pick, (0, topk - pick.shape[-1]), value=nb)
        s["num"] = blocks[..., 0].clamp(max=topk).expand(b, n, hk).int().contiguous()
        pick = torch.where(torch.arange(topk, device=DEV) < s["num"][..., None], pick, nb).sort(-1).values
        s["index"] = torch.where(pick < nb, pick, -1).int().contiguous()
    return s


# ------------------------------------------------------------------------------------------------
# One call
# ------------------------------------------------------------------------------------------------
def run(s):
    return {"ranged": _run_ranged, "cache": _run_cache, "read": _run_read, "attend": _run_attend}[s["case"]["kind"]](s)


def _run_ranged(s):
    c = s["case"]
    if not own:
        return _ranged_plain(s)
    from worldattention_amd.hsa import ranged_attention

    out, lse = ranged_attention(s["q"], s["k"], s["v"], s["ranges"], cap=c["score_cap"] or None, slopes=s["slopes"],
                                return_lse=True)
    if not s["train"]:
        return {"out": out, "lse": lse}
    names = ["q", "k", "v"] + (["slopes"] if c["slopes"] == "learnt" else [])
    grads = torch.autograd.grad(out, [s[x] for x in names], s["dout"])
    return {"out": out.detach(), "lse": lse.detach(), **{"d" + x: y for x, y in zip(names, grads)}}


def _seen(c, documents, rows):
    """Which keys the queries ``rows`` see, [rows, length], from the rules themselves."""
    j = torch.arange(c["length"], device=DEV)
    t = rows[:, None] + c["length"] - c["queries"]
    first = torch.zeros_like(j)
    mine = torch.ones((rows.numel(), c["length"]), dtype=torch.bool, device=DEV)
    if documents is not None:
        which = torch.searchsorted(documents, j.int(), right=True)
        inside = (which > 0) & (which < documents.numel())
        first = torch.where(inside, documents[(which - 1).clamp(min=0)].long(), 0)
        mine = (which[t] == which) & inside[t]
    rel_t, rel_j = t - first[t], j - first
    reach = rel_j < (rel_t // c["chunk"] + 1) * c["chunk"] if c["causal"] else torch.ones_like(mine)
    near = (j > t - c["window"]) & (c["causal"] | (j < t + c["window"])) if c["window"] else torch.ones_like(mine)
    return mine & (reach & (near | (rel_j < c["sink"])) | (rel_j < c["prefix"]))


def _ranged_plain(s):
    c = s["case"]
    b, n, m, h, hk, d = (c[x] for x in ("batch", "queries", "length", "heads", "kv_heads", "dim"))
    per, scale, train, cap = h // hk, d ** -0.5, s["train"], c["score_cap"]
    j = torch.arange(m, device=DEV)
    band = max(1, min(n, 2 ** 26 // (h * m)))
    out = torch.empty((b, n, h, d), dtype=torch.bfloat16, device=DEV)
    lse = torch.empty((b, h, n), device=DEV)
    if train:
        dq, dslope = torch.empty_like(out), torch.zeros((h,), dtype=torch.float64, device=DEV)
        dk, dv = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    for i in range(b):
        k, v = (s[x][i].float().transpose(0, 1).repeat_interleave(per, 0) for x in "kv")        # [H, M, D]
        kt = k.transpose(1, 2).contiguous()
        if train:
            vt = v.transpose(1, 2).contiguous()
            dk_sum, dv_sum = torch.zeros_like(k), torch.zeros_like(v)
        for r0 in range(0, n, band):
            rows = torch.arange(r0, min(n, r0 + band), device=DEV)
            seen = _seen(c, s["documents"], rows)
            far = (rows[:, None] + (m - n) - j).abs().float()
            q = s["q"][i, r0: r0 + band].float().transpose(0, 1).contiguous()
            x = torch.matmul(q, kt) * scale
            if cap:
                turn = torch.tanh(x / cap)
                x = cap * turn
            if s["slopes"] is not None:
                x = x - s["slopes"][:, None, None] * far
            x = torch.where(seen, x, -math.inf)
            top = x.amax(-1, keepdim=True).clamp(min=-1e30)
            p = (x - top).exp()
            total = p.sum(-1, keepdim=True)
            lse[i, :, r0: r0 + band] = (total.log() + top)[..., 0]
            p = p / total.clamp(min=1e-30)
            out[i, r0: r0 + band] = torch.matmul(p, v).transpose(0, 1).to(torch.bfloat16)
            if not train:
                continue
            do = s["dout"][i, r0: r0 + band].float().transpose(0, 1).contiguous()
            dp = torch.matmul(do, vt)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            if c["slopes"] == "learnt":
                dslope -= (ds * far).sum((1, 2), dtype=torch.float64)
            if cap:
                ds = ds * (1 - turn * turn)
            ds = ds * scale
            dq[i, r0: r0 + band] = torch.matmul(ds, k).transpose(0, 1).to(torch.bfloat16)
            dk_sum += torch.matmul(ds.transpose(1, 2).contiguous(), q)
            dv_sum += torch.matmul(p.transpose(1, 2).contiguous(), do)
        if train:
            dk[i], dv[i] = (x.view(hk, per, m, d).sum(1).transpose(0, 1).to(torch.bfloat16) for x in (dk_sum, dv_sum))
    if not train:
        return {"out": out, "lse": lse}
    grads = {"dq": dq, "dk": dk, "dv": dv, **({"dslopes": dslope.float()} if c["slopes"] == "learnt" else {})}
    return {"out": out, "lse": lse, **grads}


def _needed_scale(largest, most):
    """The smallest power of two (2^-126 at least) at which ``largest`` is at most ``most``."""
    part, power = torch.frexp(largest)
    top = math.frexp(most)
    power = power - top[1] + (part > top[0])
    return torch.ldexp(torch.ones_like(part), torch.where(largest > 0, power, -126).clamp(min=-126))


def _encode(x, codes):
    return x.round().to(torch.int8) if codes == "int8" else x.to(torch.float8_e4m3fn)


def _run_cache(s):
    c, cache = s["case"], s["cache"]
    span = c["tokens"] + c["block"] - 1
    if own:
        from worldattention_amd.hsa import kv_append_8bit, kv_read_8bit

        kv_append_8bit(cache, s["k"], s["v"], s["start"], lengths=s["counts"])
        k, v = kv_read_8bit(cache, s["first"], span)
    else:
        for x in "kv":
            _append_plain(s, x)
        k, v = (_read_plain(c, cache, x, s["first"], span).bfloat16() for x in "kv")
    return {"k": k, "v": v, "k_scale": cache["k_scale"], "v_scale": cache["v_scale"], "k_block_sums": cache["k_block_sums"]}


def _append_plain(s, x):
    """The touched blocks of every sequence, as [B, blocks, block, Hk, D] from the block that holds the first new token on."""
    c, cache = s["case"], s["cache"]
    b, n, hk, d, bs, cap, kind = (c[y] for y in ("batch", "tokens", "kv_heads", "dim", "block", "cap", "codes"))
    nt, nb = -(-(n + bs - 1) // bs), -(-cap // bs)
    at = torch.arange(b, device=DEV)[:, None]
    token = s["first"].long()[:, None] + torch.arange(nt * bs, device=DEV)
    new = token - s["start"].long()[:, None]
    count = torch.full((b, 1), n, device=DEV) if s["counts"] is None else s["counts"].long()[:, None]
    is_new = ((new >= 0) & (new < count))[..., None, None]
    is_old = (new < 0)[..., None, None]
    fresh = torch.where(is_new, s[x][at, new.clamp(0, n - 1)].float(), 0.0).view(b, nt, bs, hk, d)
    block = s["first"].long()[:, None] // bs + torch.arange(nt, device=DEV)
    touched = (is_new.view(b, nt, bs).any(-1) & (block < nb))[..., None]                            # [B, nt, 1]
    scale = cache[x + "_scale"].transpose(1, 2)
    before = torch.where(is_old.view(b, nt, bs).any(-1)[..., None], scale[at, block.clamp(max=nb - 1)], 0.0)   # [B, nt, Hk]
    now = torch.maximum(before, _needed_scale(fresh.abs().amax((2, 4)), LARGEST[kind]))
    now = torch.where(touched, now, scale[at, block.clamp(max=nb - 1)])
    held = cache[x].view(torch.uint8)[at, token.clamp(max=cap - 1)].view(CODES[kind]).float().view(b, nt, bs, hk, d)
    old = _encode(held * (before / now.clamp(min=2.0 ** -126))[:, :, None, :, None], kind)
    codes = torch.where(is_new.view(b, nt, bs, 1, 1), _encode(fresh / now[:, :, None, :, None].clamp(min=2.0 ** -126), kind).float(),
                        old.float())
    write = (touched[..., None] & (is_new | is_old).view(b, nt, bs, 1)).view(b, nt * bs) & (token < cap)
    row, col = write.nonzero(as_tuple=True)
    cache[x].view(torch.uint8)[row, token[row, col]] = _code_bytes(codes, kind).view(b, nt * bs, hk, d)[row, col]
    row, col = touched[..., 0].nonzero(as_tuple=True)
    cache[x + "_scale"][row, :, block[row, col]] = now[row, col]
    if x == "k":
        live = torch.where((is_new | is_old).view(b, nt, bs, 1, 1), codes, 0.0)
        sums = live.sum(2) * now[..., None]
        cache["k_block_sums"][row, :, block[row, col]] = sums[row, col]


def _code_bytes(codes, kind):
    return codes.to(CODES[kind]).view(torch.uint8)


def _read_plain(c, cache, x, start, n):
    """[B, n, Hk, D] in fp32; 0 behind the cache."""
    b, bs, cap = c["batch"], c["block"], c["cap"]
    at = torch.arange(b, device=DEV)[:, None]
    token = start.long()[:, None] + torch.arange(n, device=DEV)
    inside = token.clamp(max=cap - 1)
    codes = cache[x].view(torch.uint8)[at, inside].view(CODES[c["codes"]]).float()
    scale = cache[x + "_scale"].transpose(1, 2)[at, inside // bs]
    return torch.where((token < cap)[..., None, None], codes * scale[..., None], 0.0)


def _run_read(s):
    c = s["case"]
    dtype = getattr(torch, c["out"])
    if own:
        from worldattention_amd.hsa import kv_read_8bit

        k, v = kv_read_8bit(s["cache"], s["start"], c["tokens"], dtype=dtype)
    else:
        k, v = (_read_plain(c, s["cache"], x, s["start"], c["tokens"]).to(dtype) for x in "kv")
    return {"k": k, "v": v}


def _run_attend(s):
    c = s["case"]
    if own:
        from worldattention_amd.hsa import BlockSelection, attend_8bit

        chosen = BlockSelection(s["index"], s["num"]) if c["topk"] else None
        out, lse = attend_8bit(s["q"], s["cache"], s["lengths"], cap=c["score_cap"] or None, slopes=s["slopes"],
                               window=c["window"] or None, sink=c["sink"], chosen=chosen)
        return {"out": out, "lse": lse}
    b, n, h, hk, d, bs, cap = (c[x] for x in ("batch", "queries", "heads", "kv_heads", "dim", "block", "cap"))
    per = h // hk
    j = torch.arange(cap, device=DEV)
    out = torch.empty((b, n, h, d), dtype=torch.bfloat16, device=DEV)
    lse = torch.empty((b, h, n), device=DEV)
    band = max(1, min(n, 2 ** 26 // (h * cap)))
    for i in range(b):
        k, v = (s["cache"][x][i].float() * s["cache"][x + "_scale"][i].T.repeat_interleave(bs, 0)[:cap, :, None] for x in "kv")
        kt, v = k.permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()
        for r0 in range(0, n, band):
            r1 = min(n, r0 + band)
            q = s["q"][i, r0: r1].float().view(r1 - r0, hk, per, d).permute(1, 2, 0, 3).reshape(hk, per * (r1 - r0), d)
            x = torch.matmul(q, kt).view(hk, per, r1 - r0, cap) * d ** -0.5
            if c["score_cap"]:
                x = c["score_cap"] * torch.tanh(x / c["score_cap"])
            t = (s["lengths"][i].long() - n + torch.arange(r0, r1, device=DEV))[:, None]
            if c["slopes"]:
                x = x - s["slopes"].view(hk, per, 1, 1) * (t - j).float()
            seen = j <= t
            if c["window"]:
                seen &= (j > t - c["window"]) | (j < c["sink"])
            if c["topk"]:
                pick = torch.zeros((hk, r1 - r0, -(-cap // bs) + 1), dtype=torch.bool, device=DEV)
                index = s["index"][i, r0: r1].transpose(0, 1).long()
                pick.scatter_(2, torch.where(index >= 0, index, pick.shape[2] - 1), True)
                seen = seen & pick[:, :, :-1].repeat_interleave(bs, -1)[..., :cap]
                seen = seen[:, None]
            x = torch.where(seen, x, -math.inf)
            top = x.amax(-1, keepdim=True).clamp(min=-1e30)
            p = (x - top).exp()
            total = p.sum(-1, keepdim=True)
            p = p / total.clamp(min=1e-30)
            o = torch.matmul(p.view(hk, per * (r1 - r0), cap), v).view(h, r1 - r0, d)
            out[i, r0: r1] = o.transpose(0, 1).to(torch.bfloat16)
            lse[i, :, r0: r1] = (total.log() + top).view(h, r1 - r0)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------------------------------------
# What a call cannot do without
# ------------------------------------------------------------------------------------------------
def _pairs(c):
    """Pairs of a query and a key that it sees, in one sequence and head; keys that any query sees."""
    t = np.arange(c["length"] - c["queries"], c["length"])
    first, end = np.zeros_like(t), np.full_like(t, c["length"])
    docs = _documents(c)
    if docs:
        which = np.searchsorted(docs, t, side="right")
        inside = (which > 0) & (which < len(docs))
        first = np.where(inside, np.array(docs)[np.maximum(which - 1, 0)], 0)
        end = np.where(inside, np.array(docs)[np.minimum(which, len(docs) - 1)], 0)
    reach = np.minimum(end, first + ((t - first) // c["chunk"] + 1) * c["chunk"]) if c["causal"] else end
    a0, a1 = first, reach
    if c["window"]:
        a0 = np.maximum(first, t - c["window"] + 1)
        a1 = reach if c["causal"] else np.minimum(reach, t + c["window"])
    b1 = np.maximum(np.minimum(first + c["sink"], reach), np.minimum(first + c["prefix"], end))
    main = np.maximum(a1 - a0, 0)
    extra = np.maximum(b1 - first, 0) - np.maximum(np.minimum(b1, a1) - np.maximum(first, a0), 0)
    seen = np.zeros(c["length"] + 1, dtype=np.int64)
    for lo, hi in ((a0, np.maximum(a0, a1)), (first, np.maximum(first, b1))):
        np.add.at(seen, lo, 1)
        np.add.at(seen, hi, -1)
    return int((main + extra).sum()), int((np.cumsum(seen)[:-1] > 0).sum())


def work(case):
    c = case
    b, d, hk = c["batch"], c["dim"], c["kv_heads"]
    if c["kind"] == "ranged":
        pairs, keys = _pairs(c)
        rows = b * c["queries"] * c["heads"]
        if c["direction"] == "forward":
            return {"bytes": rows * (4 * d + 4) + 4 * b * keys * hk * d, "flops": 4 * b * c["heads"] * pairs * d}
        # q, k, v and dO in; O and the gradients out (the keys' whole, seen or not)
        return {"bytes": rows * (8 * d + 4) + b * hk * d * (4 * keys + 4 * c["length"]), "flops": 14 * b * c["heads"] * pairs * d}
    if c["kind"] == "cache":
        starts, counts = _written(c)
        new, bs = sum(counts), c["block"]
        back = sum(min(c["cap"], s // bs * bs + c["tokens"] + bs - 1) - s // bs * bs for s in starts)
        # new tokens in, their codes out; the blocks' earlier codes in for the keys' sums; scales and sums; what is read back
        blocks = sum(-(-(s % bs + n) // bs) for s, n in zip(starts, counts) if n)
        early = sum(s % bs for s, n in zip(starts, counts) if n)
        return {"bytes": hk * (d * (2 * 3 * new + early + 4 * blocks) + 8 * blocks + 2 * 3 * d * back), "flops": 8 * hk * d * new}
    if c["kind"] == "read":
        size = b * c["tokens"] * hk
        return {"bytes": 2 * size * d * (1 + (2 if c["out"] == "bfloat16" else 4)), "flops": 2 * size * d}
    n, bs, read, pairs = c["queries"], c["block"], 0, 0
    for length in _kv_lengths(c):
        t = np.arange(length - n, length)
        t = t[t >= 0]
        if not t.size:
            continue
        if c["topk"]:
            picked = np.minimum(t // bs + 1, c["topk"])
            tokens = (picked - 1) * bs + t % bs + 1
            pairs += int(tokens.sum())
            read += int(min(length, tokens.sum()))
        elif c["window"]:
            main = np.minimum(t + 1, c["window"])
            pairs += int((main + np.minimum(c["sink"], t + 1 - main)).sum())
            reach = min(length, length - int(t[0]) + c["window"] - 1)
            read += reach + min(c["sink"], length - reach)
        else:
            pairs += int((t + 1).sum())
            read += length
    return {"bytes": 2 * read * hk * d + b * n * c["heads"] * (4 * d + 4), "flops": 4 * pairs * c["heads"] * d}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"ranged": _exact_ranged, "cache": _exact_cache, "read": _exact_read, "attend": _exact_attend}[case["kind"]](s)


def _runs(c):
    """Every query's two runs of keys, by hand: (first, end) of its own reach and of what it always sees."""
    docs = _documents(c) or [0, c["length"]]
    out = []
    for t in range(c["length"] - c["queries"], c["length"]):
        home = [(x, y) for x, y in zip(docs, docs[1:]) if x <= t < y]
        if not home:
            out.append((0, 0, 0, 0))
            continue
        x, y = home[0]
        end = min(y, x + ((t - x) // c["chunk"] + 1) * c["chunk"]) if c["causal"] else y
        lo, hi = x, end
        if c["window"]:
            lo, hi = max(x, t - c["window"] + 1), end if c["causal"] else min(end, t + c["window"])
        out.append((lo, hi, x, max(min(x + c["sink"], end), min(x + c["prefix"], y))))
    return torch.tensor(out, device=DEV)


def _exact_ranged(s):
    c = s["case"]
    b, n, m, h, hk, d = (c[x] for x in ("batch", "queries", "length", "heads", "kv_heads", "dim"))
    f64 = dict(dtype=torch.float64, device=DEV)
    out, lse = torch.zeros((b, n, h, d), **f64), torch.zeros((b, h, n), **f64)
    grad = {"dq": torch.zeros((b, n, h, d), **f64), "dk": torch.zeros((b, m, hk, d), **f64),
            "dv": torch.zeros((b, m, hk, d), **f64), "dslopes": torch.zeros((h,), **f64)}
    runs, j = _runs(c), torch.arange(m, device=DEV)
    slopes = None if s["slopes"] is None else s["slopes"].detach().double()
    for r0 in range(0, n, 2048):
        r1 = min(n, r0 + 2048)
        w = runs[r0:r1, :, None]
        hidden = ~(((j >= w[:, 0]) & (j < w[:, 1])) | ((j >= w[:, 2]) & (j < w[:, 3])))
        far = (torch.arange(m - n + r0, m - n + r1, device=DEV)[:, None] - j).abs().double()
        for bi in range(b):
            for hi in range(h):
                q, do = (s[x][bi, r0:r1, hi].detach().double() if x in s else None for x in ("q", "dout"))
                k, v = (s[x][bi, :, hi // (h // hk)].detach().double() for x in "kv")
                logit = (q @ k.T) / math.sqrt(d)
                if c["score_cap"]:
                    bent = torch.tanh(logit / c["score_cap"])
                    logit = bent * c["score_cap"]
                if slopes is not None:
                    logit = logit.sub_(slopes[hi] * far)
                logit.masked_fill_(hidden, -math.inf)
                total = torch.logsumexp(logit, -1)
                lse[bi, hi, r0:r1] = total
                p = logit.sub_(total.clamp(min=-1e300)[:, None]).exp_()
                out[bi, r0:r1, hi] = p @ v
                if not s["train"]:
                    continue
                grad["dv"][bi, :, hi // (h // hk)] += p.T @ do
                ds = do @ v.T
                ds = (ds - (do * out[bi, r0:r1, hi]).sum(-1, keepdim=True)) * p
                grad["dslopes"][hi] -= (ds * far).sum()
                if c["score_cap"]:
                    ds = ds * (1 - bent ** 2)
                ds /= math.sqrt(d)
                grad["dq"][bi, r0:r1, hi] = ds @ k
                grad["dk"][bi, :, hi // (h // hk)] += ds.T @ q
    if not s["train"]:
        return {"out": out, "lse": lse}
    if c["slopes"] != "learnt":
        del grad["dslopes"]
    return {"out": out, "lse": lse, **grad}


def _rounded(x, kind):
    """``x`` to the nearest value that a code stands for, ties to the even code."""
    if kind == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _power(largest, kind):
    """As a Python float: the smallest power of two at which ``largest`` fits the codes."""
    scale = 2.0 ** -126
    while largest > LARGEST[kind] * scale:
        scale *= 2.0
    return scale


def _exact_cache(s):
    """Sequence by sequence and block by block."""
    c, cache = s["case"], s["cache"]
    b, n, hk, d, bs, cap, kind = (c[x] for x in ("batch", "tokens", "kv_heads", "dim", "block", "cap", "codes"))
    if b * hk * -(-(n + bs - 1) // bs) > 4096:
        return None
    starts, counts = _written(c)
    span = n + bs - 1
    scales = {x: cache[x + "_scale"].double() for x in "kv"}
    sums = cache["k_block_sums"].double()
    read = {x: torch.zeros((b, span, hk, d), dtype=torch.float64, device=DEV) for x in "kv"}
    for x in "kv":
        for i, (start, count) in enumerate(zip(starts, counts)):
            first = start // bs * bs
            codes = cache[x][i].to(torch.float64)
            for block in range(first // bs, -(-(start + count) // bs) if count else first // bs):
                lo, hi = block * bs, min((block + 1) * bs, start + count)
                fresh = s[x][i, max(lo, start) - start: hi - start].double()
                need = fresh.abs().amax((0, 2)).tolist()
                for e in range(hk):
                    held = float(scales[x][i, e, block]) if lo < start else 0.0
                    scale = max(held, _power(need[e], kind))
                    if lo < start:
                        codes[lo:start, e] = _rounded(codes[lo:start, e] * (held / scale), kind)
                    codes[max(lo, start): hi, e] = _rounded(fresh[:, e] / scale, kind)
                    scales[x][i, e, block] = scale
                    if x == "k":
                        sums[i, e, block] = codes[lo:hi, e].sum(0) * scale
            size = min(span, cap - first)
            block = torch.arange(first, first + size, device=DEV) // bs
            read[x][i, :size] = codes[first: first + size] * scales[x][i, :, block].T[..., None]
    return {"k": read["k"], "v": read["v"], "k_scale": scales["k"], "v_scale": scales["v"], "k_block_sums": sums}


def _exact_read(s):
    c, out = s["case"], {}
    starts = s["start"].tolist()
    for x in "kv":
        rows = []
        for i, start in enumerate(starts):
            block = torch.arange(start, start + c["tokens"], device=DEV) // c["block"]
            rows.append(s["cache"][x][i, start: start + c["tokens"]].to(torch.float64)
                        * s["cache"][x + "_scale"][i].double()[:, block].T[..., None])
        out[x] = torch.stack(rows)
    return out


def _exact_attend(s):
    """Each sequence and head by itself over the tokens it holds."""
    c = s["case"]
    b, n, h, hk, d, bs = (c[x] for x in ("batch", "queries", "heads", "kv_heads", "dim", "block"))
    out = torch.zeros((b, n, h, d), dtype=torch.float64, device=DEV)
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64, device=DEV)
    for bi, length in enumerate(_kv_lengths(c)):
        if not length:
            continue
        j = torch.arange(length, device=DEV)
        t = torch.arange(length - n, length, device=DEV)[:, None]
        for e in range(hk):
            k, v = (s["cache"][x][bi, :length, e].to(torch.float64) * s["cache"][x + "_scale"][bi, e].double()[j // bs][:, None]
                    for x in "kv")
            hidden = j > t
            if c["window"]:
                hidden |= (j + c["window"] <= t) & (j >= c["sink"])
            if c["topk"]:
                hidden |= ~(s["index"][bi, :, e, :, None] == j // bs).any(1)
            for hi in range(e * (h // hk), (e + 1) * (h // hk)):
                logit = s["q"][bi, :, hi].double() @ k.T / math.sqrt(d)
                if c["score_cap"]:
                    logit = torch.tanh(logit / c["score_cap"]) * c["score_cap"]
                if c["slopes"]:
                    logit = logit - s["slopes"][hi].double() * (t - j)
                logit = logit.masked_fill(hidden, -math.inf)
                lse[bi, hi] = torch.logsumexp(logit, -1)
                out[bi, :, hi] = (logit - lse[bi, hi].clamp(min=-1e300)[:, None]).exp() @ v
    return {"out": out, "lse": lse}
