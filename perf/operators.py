"""The token-by-token operators: rotary positions with several axes, linear attention with a decay for
each head (prompts, training and single tokens) and attention of single queries over the key blocks
that a score selects from a cache.

They serve a causal model that reads and writes its KV cache token by token: every layer rotates its
queries and keys (``rope``), its linear heads carry a decayed state (``decay``, ``step``) and its
sparse heads read a few blocks of the cache (``select``). Each kind of case is one call of such a
layer; the training kinds return the gradients too.
"""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # One new token of each of 16 sequences, far into them: launches and host time decide it.
        _rope("rope_step", "forward", "bfloat16", 16, 1, 32, 8, 128, 3, True, "far"),
        # Training on one chunk of a video (3 frames of 30 x 52 latent tokens), forward and backward.
        _rope("rope_train_chunk", "train", "bfloat16", 1, 4680, 12, 12, 128, 3, True, "grid"),
        # A whole window of 21 frames with 40 heads as a prompt: all memory traffic.
        _rope("rope_window_40heads", "forward", "bfloat16", 1, 32760, 40, 40, 128, 3, True, "grid"),
        # One token of one sequence through 12 linear heads: latency.
        dict(name="step_one", kind="step", dtype="bfloat16", batch=1, heads=12, dim=128),
        # One token of each of 64 sequences: the states are read and written once.
        dict(name="step_batch", kind="step", dtype="bfloat16", batch=64, heads=16, dim=128),
        # A padded batch of prompts whose states go on into the decoding.
        _decay("decay_prompt_ragged", "forward", "bfloat16", 4, 5003, 12, 128, True),
        # The whole window of 21 frames as one causal prompt.
        _decay("decay_prompt_window", "forward", "bfloat16", 1, 32760, 12, 128, False),
        # A training step over the same length: all gradients, the decays' and the initial state's too.
        _decay("decay_train_window", "train", "bfloat16", 1, 32760, 12, 128, False),
        # A small model in fp32 with 64-channel heads on an odd length.
        _decay("decay_train_fp32", "train", "float32", 2, 1111, 4, 64, True),
        # One token of one sequence with shared key heads over a cache of 4 K tokens: latency.
        _select("select_step", "bfloat16", 1, 1, 32, 8, 128, 4096, 64, 16, False),
        # One token each of a served batch of ragged sequences.
        _select("select_batch", "bfloat16", 32, 1, 32, 8, 128, 32768, 64, 32, True),
        # A chunk of a long prompt: every token selects its own blocks.
        _select("select_prompt", "bfloat16", 1, 1024, 32, 8, 128, 16384, 64, 16, False),
    ]


def _rope(name, direction, dtype, batch, length, heads, kv_heads, dim, axes, interleaved, where):
    return _named(name, dict(kind="rope", direction=direction, dtype=dtype, batch=batch, length=length, heads=heads,
                             kv_heads=kv_heads, dim=dim, axes=axes, interleaved=interleaved, where=where))


def _decay(name, direction, dtype, batch, length, heads, dim, ragged):
    return _named(name, dict(kind="decay", direction=direction, dtype=dtype, batch=batch, length=length, heads=heads,
                             dim=dim, ragged=ragged))


def _select(name, dtype, batch, queries, heads, kv_heads, dim, cap, block, topk, ragged):
    return _named(name, dict(kind="select", dtype=dtype, batch=batch, queries=queries, heads=heads, kv_heads=kv_heads,
                             dim=dim, cap=cap, block=block, topk=topk, sink=1, local=2, ragged=ragged))


def _named(name, case):
    return case if name is None else dict(name=name, **case)


def _spread(rng, low, high):
    """A whole number, even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["rope", "step", "decay", "decay", "select", "select"])
    if kind == "rope":
        heads = rng.randint(1, 40)
        kv_heads = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
        batch = _spread(rng, 1, 16)
        return _rope(None, rng.choice(["forward", "train"]), rng.choice(["bfloat16", "bfloat16", "float32"]), batch,
                     _spread(rng, 1, min(32760, 600000 // (heads * batch))), heads, kv_heads,
                     rng.choice([64, 96, 128]), rng.randint(1, 3), rng.random() < 0.5, rng.choice(["far", "grid"]))
    if kind == "step":
        heads = rng.randint(1, 40)
        return dict(kind="step", dtype=rng.choice(["bfloat16", "float32"]), batch=_spread(rng, 1, 1024 // heads),
                    heads=heads, dim=rng.choice([64, 80, 128]))
    if kind == "decay":
        direction = rng.choice(["forward", "train"])
        heads, batch = rng.randint(1, 16), rng.randint(1, 4)
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        most = min(32760, (200000 if dtype == "bfloat16" else 50000) // (heads * batch))
        return _decay(None, direction, dtype, batch, _spread(rng, 1, most), heads, rng.choice([64, 128]),
                      rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    batch, queries = (_spread(rng, 1, 32), rng.randint(1, 4)) if rng.random() < 0.6 else (1, _spread(rng, 5, 1024))
    block = rng.choice([64, 128])
    topk = rng.randint(4, 32 if queries <= 4 else 16 * 64 // block)
    cap = _spread(rng, 2 * block, max(4 * block, min(131072, 8 * 1048576 // (batch * kv_heads))))
    return _select(None, "bfloat16", batch, min(queries, cap // 2), heads, kv_heads, rng.choice([64, 128]), cap, block,
                   topk, batch > 1)


def _lengths(case):
    """The sequences' lengths: all of them whole, or spread from the whole one to short ones (one of them empty in a padded
    batch of prompts, one shorter than its queries in a batch over a cache)."""
    batch, full = case["batch"], case.get("cap", case.get("length"))
    if not case["ragged"]:
        return [full] * batch
    return [max(0, full - (full * b) // (batch - 1)) if batch > 1 else full for b in range(batch)]


# ------------------------------------------------------------------------------------------------
# What a program has in hand before the call
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"rope": _prepare_rope, "step": _prepare_step, "decay": _prepare_decay, "select": _prepare_select}[
        case["kind"]](case, g)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _prepare_rope(case, g):
    dt, b, n, d = DTYPES[case["dtype"]], case["batch"], case["length"], case["dim"]
    train = case["direction"] == "train"
    half = d // 2
    third = half // 3
    sections = {1: (half,), 2: (half - third, third), 3: (half - 2 * third, third, third)}[case["axes"]]
    inv = torch.cat([10000.0 ** -(torch.arange(s, device=DEV, dtype=torch.float64) / s) for s in sections])
    t = torch.arange(n, device=DEV)
    if case["where"] == "grid":  # frames of 30 x 52 tokens, the batch at the same places
        pos = torch.stack([t // 1560, t // 52 % 30, t % 52][: case["axes"]], dim=-1)
    else:  # tokens of sequences of their own, up to a million tokens in
        first = torch.randint(0, 1000000, (b, 1, case["axes"]), generator=g, device=DEV)
        pos = first + t[:, None]
    s = dict(case=case, pos=pos, inv=inv, sections=sections, train=train)
    for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
        s[name] = _normal(g, (b, n, heads, d), dt).requires_grad_(train)
        if train:
            s["d" + name] = _normal(g, (b, n, heads, d), dt)
    return s


def _log_decay(case, g):
    """Decays whose memory spans from 8 to 1024 tokens over the heads."""
    h = torch.arange(case["heads"], device=DEV, dtype=torch.float32)
    jitter = 0.5 * torch.rand(case["heads"], generator=g, device=DEV)
    return -torch.exp2(-(3.0 + 6.5 * h / max(1, case["heads"] - 1)) - jitter)


def _prepare_step(case, g):
    dt, b, h, d = DTYPES[case["dtype"]], case["batch"], case["heads"], case["dim"]
    q, k, v = (_normal(g, (b, 1, h, d), dt) for _ in range(3))
    return dict(case=case, q=q, k=k, v=v, log_decay=_log_decay(case, g),
                state=_normal(g, (b, h, d, d), torch.float32))


def _prepare_decay(case, g):
    dt, b, n, h, d = DTYPES[case["dtype"]], case["batch"], case["length"], case["heads"], case["dim"]
    train = case["direction"] == "train"
    q, k, v = (_normal(g, (b, n, h, d), dt) for _ in range(3))
    s = dict(case=case, q=q, k=k, v=v, log_decay=_log_decay(case, g), train=train,
             initial=_normal(g, (b, h, d, d), torch.float32) if train else None,
             lengths=torch.tensor(_lengths(case), dtype=torch.int32, device=DEV) if case["ragged"] else None)
    if train:
        for name in ("q", "k", "v", "log_decay", "initial"):
            s[name].requires_grad_(True)
        s["dout"] = _normal(g, (b, n, h, d), dt)
        s["dfinal"] = _normal(g, (b, h, d, d), torch.float32)
    return s


def _prepare_select(case, g):
    dt, b, hk, d, cap, bs = (DTYPES[case["dtype"]], case["batch"], case["kv_heads"], case["dim"], case["cap"],
                             case["block"])
    nb = -(-cap // bs)
    q = _normal(g, (b, case["queries"], case["heads"], d), dt)
    # keys of a block share a direction, as neighbouring tokens do
    k = torch.randn((b, cap, hk, d), generator=g, device=DEV, dtype=dt)
    topic = torch.randn((b, nb, hk, d), generator=g, device=DEV, dtype=dt) * 0.5
    k += topic.repeat_interleave(bs, dim=1)[:, :cap]
    v = torch.randn((b, cap, hk, d), generator=g, device=DEV, dtype=dt)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    # the sums of every block, as the cache keeps them beside its keys
    sums = torch.zeros((b, nb, hk, d), device=DEV)
    whole = cap // bs
    sums[:, :whole] = k[:, : whole * bs].reshape(b, whole, bs, hk, d).sum(dim=2, dtype=torch.float32)
    if whole < nb:
        sums[:, whole] = k[:, whole * bs:].sum(dim=1, dtype=torch.float32)
    cache = {"k": k, "v": v, "k_block_sums": sums.transpose(1, 2).contiguous(), "k_block_sums_block_size": bs}
    return dict(case=case, q=q, cache=cache, lengths=lengths)


# ------------------------------------------------------------------------------------------------
# One call
# ------------------------------------------------------------------------------------------------
def run(s):
    return {"rope": _run_rope, "step": _run_step, "decay": _run_decay, "select": _run_select}[s["case"]["kind"]](s)


def _run_rope(s):
    if own:
        from worldattention_amd.hsa import rope_axes

        q, k = rope_axes(s["q"], s["pos"], s["inv"], s["sections"], k=s["k"], interleaved=s["case"]["interleaved"])
    else:
        axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=DEV),
                                       torch.tensor(s["sections"], device=DEV), output_size=s["inv"].numel())
        angle = s["pos"].double()[..., axis] * s["inv"]
        turn = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
        q, k = (_rotate(s[name], *turn, s["case"]["interleaved"]) for name in ("q", "k"))
    if not s["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _rotate(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    f = x[..., : 2 * pairs].float()
    even, odd = (f[..., 0::2], f[..., 1::2]) if interleaved else (f[..., :pairs], f[..., pairs:])
    re, im = even * cos - odd * sin, even * sin + odd * cos
    turned = torch.stack((re, im), dim=-1).flatten(-2) if interleaved else torch.cat((re, im), dim=-1)
    return torch.cat((turned.to(x.dtype), x[..., 2 * pairs:]), dim=-1)


def _run_step(s):
    if own:
        from worldattention_amd.hsa import decay_linear_step

        return {"out": decay_linear_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"]), "state": s["state"]}
    q, k, v = (s[name][:, 0].float() for name in ("q", "k", "v"))
    s["state"].mul_(s["log_decay"].exp()[:, None, None]).add_(k.unsqueeze(-1) * v.unsqueeze(-2))
    out = torch.matmul(q.unsqueeze(-2), s["state"]).squeeze(-2) * s["case"]["dim"] ** -0.5
    return {"out": out.unsqueeze(1).to(s["q"].dtype), "state": s["state"]}


def _run_decay(s):
    if own:
        from worldattention_amd.hsa import decay_linear_attention

        out, final = decay_linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["initial"],
                                            lengths=s["lengths"])
    else:
        out, final = _decay_chunks(s["q"], s["k"], s["v"], s["log_decay"], s["initial"], s["lengths"])
    if not s["train"]:
        return {"out": out, "state": final}
    names = ("q", "k", "v", "log_decay", "initial")
    grads = torch.autograd.grad((out, final), [s[n] for n in names], (s["dout"], s["dfinal"]))
    return {"out": out.detach(), "state": final.detach(), **{"d" + n: d for n, d in zip(names, grads)}}


def _decay_chunks(q, k, v, log_decay, initial, lengths):
    """Chunks of 128 tokens: products inside a chunk, states between chunks."""
    b, n, h, d = q.shape
    c = 128
    nc = -(-n // c)
    t = torch.arange(n, device=DEV)
    end = lengths.long()[:, None] if lengths is not None else torch.full((b, 1), n, device=DEV)
    real = (t < end)[..., None, None]

    def split(x):  # [B, H, chunks, C, D]
        x = torch.where(real, x.float(), 0.0)
        return torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nc * c - n)).view(b, nc, c, h, d).permute(0, 3, 1, 2, 4)

    def power(steps):  # decay ** steps for [...] whole steps, 0 where they are negative: [H, ...]
        g = log_decay.double().view(h, *[1] * steps.dim())
        return torch.where(steps >= 0, (g * steps.clamp(min=0)).exp(), 0.0).float()

    qc, kc, vc = split(q), split(k), split(v)
    i, m = torch.arange(c, device=DEV), torch.arange(nc, device=DEV)
    inside = torch.matmul(qc, kc.transpose(-1, -2).contiguous()) * power(i[:, None] - i)[:, None]
    out = torch.matmul(inside, vc)
    local = torch.matmul((kc * power(c - 1 - i)[:, None, :, None]).transpose(-1, -2).contiguous(), vc)
    before = torch.matmul(power((m[:, None] - 1 - m) * c), local.flatten(-2)).view(b, h, nc, d, d)
    if initial is not None:
        before = before + power(m * c)[..., None, None] * initial[:, :, None]
    out = out + torch.matmul(qc * power(i + 1)[:, None, :, None], before)
    out = (out * d ** -0.5).permute(0, 2, 3, 1, 4).reshape(b, nc * c, h, d)[:, :n]
    kept = power(end - 1 - t).transpose(0, 1)[..., None]  # [B, H, L, 1]
    kf, vf = (torch.where(real, x.float(), 0.0).transpose(1, 2) for x in (k, v))
    final = torch.matmul((kf * kept).transpose(-1, -2).contiguous(), vf.contiguous())
    if initial is not None:
        final = final + power(end[:, 0]).transpose(0, 1)[..., None, None] * initial
    return torch.where(real, out, 0.0).to(q.dtype), final


def _run_select(s):
    c = s["case"]
    if own:
        from worldattention_amd.hsa import attend_selected

        out, lse, chosen = attend_selected(s["q"], s["cache"], s["lengths"], topk=c["topk"], sink_blocks=c["sink"],
                                           local_blocks=c["local"])
        return {"out": out, "lse": lse, "index": chosen.index, "num": chosen.num}
    index, num, seen = _choose(s["q"], s["cache"]["k_block_sums"], s["lengths"], c)
    out, lse = _attend(s["q"], s["cache"]["k"], s["cache"]["v"], index, seen, c["block"])
    return {"out": out, "lse": lse, "index": index, "num": num}


def _choose(q, sums, lengths, c):
    b, n, h, d = q.shape
    hk, nb = sums.shape[1:3]
    seen = (lengths.long()[:, None] - n + 1 + torch.arange(n, device=DEV)).clamp(min=0)  # tokens, [B, n]
    blocks = (seen + c["block"] - 1) // c["block"]
    group = q.double().view(b, n, hk, h // hk, d).sum(3)
    score = torch.matmul(group.transpose(1, 2), sums.double().transpose(-1, -2)).transpose(1, 2)  # [B, n, Hk, blocks]
    j = torch.arange(nb, device=DEV)
    vis = blocks[..., None, None]
    score = torch.where((j < c["sink"]) | (j >= vis - c["local"]), math.inf, score)
    score = torch.where(j < vis, score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., : c["topk"]]
    order = torch.nn.functional.pad(order, (0, c["topk"] - order.shape[-1]), value=nb)
    num = blocks.clamp(max=c["topk"])[..., None].expand(b, n, hk)
    order = torch.where(torch.arange(c["topk"], device=DEV) < num[..., None], order, nb).sort(-1).values
    return torch.where(order < nb, order, -1).int(), num.int(), seen


def _attend(q, k, v, index, seen, bs):
    b, n, h, d = q.shape
    cap, hk = k.shape[1:3]
    token = (index.long()[..., None] * bs + torch.arange(bs, device=DEV)).flatten(3)  # [B, n, Hk, picked tokens]
    live = (index >= 0).repeat_interleave(bs, dim=-1) & (token < seen[..., None, None])
    token = token.clamp(0, cap - 1)
    at = torch.arange(b, device=DEV)[:, None, None, None], torch.arange(hk, device=DEV)[:, None]
    keys, values = (torch.where(live[..., None], x[at[0], token, at[1]].float(), 0.0) for x in (k, v))
    logits = torch.matmul(q.float().view(b, n, hk, h // hk, d), keys.transpose(-1, -2)) * d ** -0.5
    logits = torch.where(live[..., None, :], logits, -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (logits - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / total.clamp(min=1e-30)
    lse = (total.log() + top).squeeze(-1)
    return out.reshape(b, n, h, d).to(q.dtype), lse.reshape(b, n, h).transpose(1, 2).contiguous()


# ------------------------------------------------------------------------------------------------
# What a call cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    es = 2 if case["dtype"] == "bfloat16" else 4
    b, d = case["batch"], case["dim"]
    if case["kind"] == "rope":
        tokens, heads = b * case["length"], case["heads"] + case["kv_heads"]
        passes = 2 if case["direction"] == "train" else 1
        places = tokens if case["where"] == "far" else case["length"]
        return {"bytes": passes * (2 * tokens * heads * d * es + places * case["axes"] * 8),
                "flops": passes * 3 * tokens * heads * d}
    if case["kind"] == "step":
        rows = b * case["heads"]
        return {"bytes": rows * (8 * d * d + 4 * d * es), "flops": rows * 5 * d * d}
    if case["kind"] == "decay":
        rows = sum(_lengths(case)) * case["heads"]
        states = b * case["heads"] * d * d * 4
        if case["direction"] == "forward":
            return {"bytes": 3 * rows * d * es + b * case["length"] * case["heads"] * d * es + states,
                    "flops": 4 * rows * d * d}
        # q, k, v and dO in, O and three gradients out; the states both ways with their gradients
        return {"bytes": 4 * rows * d * es + 4 * b * case["length"] * case["heads"] * d * es + 4 * states,
                "flops": 14 * rows * d * d}
    n, bs, hk = case["queries"], case["block"], case["kv_heads"]
    size, flops = b * n * case["heads"] * (2 * d * es + 4), 0
    for length in _lengths(case):
        blocks = -(-length // bs)
        picked = min(blocks, case["topk"]) * bs
        size += hk * d * (4 * blocks + 2 * es * min(length, n * picked)) + n * hk * 4 * (case["topk"] + 1)
        flops += n * (2 * hk * blocks * d + 4 * case["heads"] * min(length, picked) * d)
    return {"bytes": size, "flops": flops}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rope": _exact_rope, "step": _exact_step, "decay": _exact_decay, "select": _exact_select}[
            case["kind"]](s)


def _exact_rope(s):
    """Pairs as complex numbers times exp(i angle); the gradient times its conjugate."""
    out, first = {}, 0
    phase = torch.empty((*s["pos"].shape[:-1], s["inv"].numel()), dtype=torch.float64, device=DEV)
    for axis, size in enumerate(s["sections"]):
        phase[..., first: first + size] = s["pos"][..., axis: axis + 1].double() * s["inv"][first: first + size]
        first += size
    turn = torch.polar(torch.ones_like(phase), phase).unsqueeze(-2)
    for name in ("q", "k", "dq", "dk") if s["train"] else ("q", "k"):
        x = s[name].detach().double()
        rest = x[..., 2 * first:]
        x = x[..., : 2 * first]
        x = x.unflatten(-1, (first, 2)) if s["case"]["interleaved"] else x.unflatten(-1, (2, first)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(x.contiguous()) * (turn.conj() if name[0] == "d" else turn))
        z = z if s["case"]["interleaved"] else z.transpose(-1, -2)
        out[name] = torch.cat((z.flatten(-2), rest), dim=-1)
    return out


def _exact_step(s):
    q, k, v = (s[name][:, 0].double() for name in ("q", "k", "v"))
    state = s["state"].double() * torch.exp(s["log_decay"].double()).view(1, -1, 1, 1)
    state = state + torch.einsum("bhd,bhe->bhde", k, v)
    out = torch.einsum("bhd,bhde->bhe", q, state) / math.sqrt(s["case"]["dim"])
    return {"out": out.unsqueeze(1), "state": state}


def _exact_decay(s):
    """The sums over all pairs of tokens j <= i, a band of rows at a time, and their derivatives written out."""
    c = s["case"]
    b, n, h, d = (c[x] for x in ("batch", "length", "heads", "dim"))
    train, scale = s["train"], d ** -0.5
    f64 = dict(dtype=torch.float64, device=DEV)
    out, final = torch.zeros((b, n, h, d), **f64), torch.zeros((b, h, d, d), **f64)
    grad = {x: torch.zeros((b, n, h, d), **f64) for x in "qkv"}
    dlog, dinit = torch.zeros(h, **f64), torch.zeros((b, h, d, d), **f64)
    for bi, length in enumerate(_lengths(c)):
        for hi in range(h):
            g = s["log_decay"][hi].detach().double()
            q, k, v = (s[x][bi, :length, hi].detach().double() for x in "qkv")
            t = torch.arange(length, **f64)
            w_end = torch.exp(g * (length - 1 - t))[:, None]
            final[bi, hi] = (k * w_end).T @ v
            if train:
                do, df = s["dout"][bi, :length, hi].double(), s["dfinal"][bi, hi].double()
                init = s["initial"][bi, hi].detach().double()
                w_start = torch.exp(g * (t + 1))[:, None]
                whole = torch.exp(g * length)
                final[bi, hi] += whole * init
                out[bi, :length, hi] = scale * w_start * (q @ init)
                kd, vd = k @ df, v @ df.T
                grad["q"][bi, :length, hi] = scale * w_start * (do @ init.T)
                grad["k"][bi, :length, hi] = w_end * vd
                grad["v"][bi, :length, hi] = w_end * kd
                dinit[bi, hi] = scale * (q * w_start).T @ do + whole * df
                dlog[hi] += (scale * (w_start * (t + 1)[:, None] * (q @ init) * do).sum()
                             + (w_end * (length - 1 - t)[:, None] * kd * v).sum() + length * whole * (init * df).sum())
            for r0 in range(0, length, 2048):
                r1 = min(length, r0 + 2048)
                lag = t[r0:r1, None] - t[None, :r1]
                decay = torch.where(lag >= 0, torch.exp(g * lag.clamp(min=0)), 0.0) * scale
                a = q[r0:r1] @ k[:r1].T * decay
                out[bi, r0:r1, hi] += a @ v[:r1]
                if train:
                    e = do[r0:r1] @ v[:r1].T
                    dlog[hi] += (a * e * lag).sum()
                    e *= decay
                    grad["q"][bi, r0:r1, hi] += e @ k[:r1]
                    grad["k"][bi, :r1, hi] += e.T @ q[r0:r1]
                    grad["v"][bi, :r1, hi] += a.T @ do[r0:r1]
    if not train:
        return {"out": out, "state": final}
    return {"out": out, "state": final, "dq": grad["q"], "dk": grad["k"], "dv": grad["v"], "dlog_decay": dlog,
            "dinitial": dinit}


def _exact_select(s):
    """Each sequence and key head by itself: ranks by counting, a softmax over the whole cache under a mask."""
    c = s["case"]
    b, n, h, hk, d, bs, topk = (c[x] for x in ("batch", "queries", "heads", "kv_heads", "dim", "block", "topk"))
    per = h // hk
    out = torch.zeros((b, n, h, d), dtype=torch.float64, device=DEV)
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64, device=DEV)
    index = torch.full((b, n, hk, topk), -1, dtype=torch.int32, device=DEV)
    num = torch.zeros((b, n, hk), dtype=torch.int32, device=DEV)
    for bi, length in enumerate(_lengths(c)):
        blocks = -(-length // bs)
        if not blocks:
            continue
        see = (length - n + 1 + torch.arange(n, device=DEV)).clamp(min=0)[:, None]
        nvis = (see + bs - 1) // bs
        j = torch.arange(blocks, device=DEV)
        t = torch.arange(length, device=DEV)
        for hi in range(hk):
            q = s["q"][bi, :, hi * per: (hi + 1) * per].double()
            score = q.sum(1) @ s["cache"]["k_block_sums"][bi, hi, :blocks].double().T
            forced = (j < c["sink"]) | (j >= nvis - c["local"])
            forced &= j < nvis
            middle = (j < nvis) & ~forced
            room = topk - forced.sum(-1, keepdim=True)
            pick = forced.clone()
            for i0 in range(0, n, 64):
                sc, mid = score[i0: i0 + 64], middle[i0: i0 + 64]
                ahead = (sc[:, None, :] > sc[:, :, None]) | ((sc[:, None, :] == sc[:, :, None]) & (j < j[:, None]))
                rank = (ahead & mid[:, None, :]).sum(-1)
                pick[i0: i0 + 64] |= mid & (rank < room[i0: i0 + 64])
            num[bi, :, hi] = pick.sum(-1)
            place = pick.cumsum(-1) - 1
            row, col = pick.nonzero(as_tuple=True)
            index[bi, row, hi, place[row, col]] = col.int()
            live = pick[:, j.repeat_interleave(bs)[:length]] & (t < see)
            keys, values = (s["cache"][x][bi, :length, hi].double() for x in ("k", "v"))
            for e in range(per):
                logit = torch.where(live, q[:, e] @ keys.T / math.sqrt(d), -math.inf)
                total = torch.logsumexp(logit, dim=-1)
                p = torch.where(live, torch.exp(logit - total.clamp(min=-1e300)[:, None]), 0.0)
                out[bi, :, hi * per + e] = p @ values
                lse[bi, hi * per + e] = total
    return {"out": out, "lse": lse, "index": index, "num": num}
