"""Plain 64-bit forms of the token-by-token operators: rotary positions with several axes, linear
attention with a decay for each head (as the recurrence it is), block selection and attention over
the selected blocks of a cache. Written from the definitions, token by token, on any device."""
from __future__ import annotations

import math

import torch


def rope_axes(x, positions, inv_freq, sections, *, interleaved=True):
    """``x`` ``[B, L, H, D]`` rotated in fp64; differentiable."""
    pairs = sum(sections)
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    pos = positions if positions.dim() == 3 else positions.expand(x.shape[0], *positions.shape)
    angle = (pos[..., axis].double() * inv_freq.double())[:, :, None]
    c, s = angle.cos(), angle.sin()
    f = x.double()
    re, im = (f[..., 0:2 * pairs:2], f[..., 1:2 * pairs:2]) if interleaved else (f[..., :pairs], f[..., pairs:2 * pairs])
    out = re * c - im * s, re * s + im * c
    turned = torch.stack(out, -1).flatten(-2) if interleaved else torch.cat(out, -1)
    return torch.cat((turned, f[..., 2 * pairs:]), -1)


def decay_linear_attention(q, k, v, log_decay, *, initial_state=None, lengths=None, scale=None):
    """``S_t = exp(log_decay) S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t``, one token after the other.
    Returns ``(out, final state)`` in fp64; differentiable. Rows from ``lengths[b]`` on are 0."""
    b, n, h, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    lam = log_decay.double().clamp(min=-1e30).exp().view(1, h, 1, 1)
    state = q.new_zeros((b, h, d, v.shape[-1]), dtype=torch.float64) if initial_state is None else initial_state.double()
    rows = []
    for t in range(n):
        live = torch.ones(b, dtype=torch.bool, device=q.device) if lengths is None else lengths > t
        live = live.view(b, 1, 1, 1)
        kt, vt, qt = (torch.where(live[..., 0], x[:, t].double(), 0.0) for x in (k, v, q))
        new = lam * state + kt[..., :, None] * vt[..., None, :]
        state = torch.where(live, new, state)
        rows.append(torch.where(live[..., 0], scale * (qt[..., None, :] @ state)[..., 0, :], 0.0))
    return (torch.stack(rows, 1) if rows else v.new_zeros(v.shape, dtype=torch.float64)), state


def select_key_blocks(q, k_block_sums, kv_len, *, block_size, topk, sink_blocks=1, local_blocks=1):
    """``(index [B, n, Hk, topk], num [B, n, Hk])`` on the host: query ``i`` of ``n`` sits at token
    ``kv_len - n + i`` and sees the blocks up to its own."""
    b, n, h, d = q.shape
    hk = k_block_sums.shape[1]
    index = torch.full((b, n, hk, topk), -1, dtype=torch.int32)
    num = torch.zeros((b, n, hk), dtype=torch.int32)
    scores = torch.matmul(q.double().cpu().view(b, n, hk, h // hk, d).sum(3).transpose(1, 2),
                          k_block_sums.double().cpu().transpose(-1, -2))
    for bi in range(b):
        for i in range(n):
            seen = max(0, int(kv_len[bi]) - n + i + 1)
            blocks = -(-seen // block_size)
            forced = {j for j in range(blocks) if j < sink_blocks or j >= blocks - local_blocks}
            for hi in range(hk):
                row = scores[bi, hi, i].tolist()
                key = lambda j: (0 if math.isnan(row[j]) else 1, -row[j], j)  # noqa: E731  NaN first, as the largest
                rest = sorted((j for j in range(blocks) if j not in forced), key=key)
                pick = sorted(forced | set(rest[:topk - len(forced)]))
                num[bi, i, hi] = len(pick)
                index[bi, i, hi, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return index, num


def selected_attention(q, k, v, index, num, kv_len, *, block_size, scale=None):
    """``(out [B, n, H, D], lse [B, H, n])`` in fp64 on the host over the first ``num`` listed blocks' visible
    tokens (ids that name no visible block add nothing; one listed twice counts twice)."""
    b, n, h, d = q.shape
    hk = k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros((b, n, h, d), dtype=torch.float64)
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64)
    q, k, v, index, num = q.double().cpu(), k.cpu(), v.cpu(), index.cpu(), num.cpu()
    for bi in range(b):
        for i in range(n):
            seen = max(0, min(int(kv_len[bi]), k.shape[1]) - n + i + 1)
            for hi in range(hk):
                ids = [int(j) for j in index[bi, i, hi, :int(num[bi, i, hi])]]
                tok = [t for j in ids if j >= 0 for t in range(j * block_size, min(seen, (j + 1) * block_size))]
                if not tok:
                    continue
                keys, values = k[bi, tok, hi].double(), v[bi, tok, hi].double()
                for g in range(hi * (h // hk), (hi + 1) * (h // hk)):
                    logit = scale * keys @ q[bi, i, g]
                    lse[bi, g, i] = torch.logsumexp(logit, 0)
                    out[bi, i, g] = torch.softmax(logit, 0) @ values
    return out, lse
