"""Plain 64-bit forms of the ranged attention: which keys a row sees, by the rules token by token, and the
attention itself under a mask of booleans. Written from the definitions, on any device; differentiable."""
from __future__ import annotations

import math

import torch


def seen(batch, q_len, k_len, *, causal=True, chunk=1, window=None, sink=0, prefix=0, documents=None, lengths=None, kv_len=None):
    """bool ``[B, q_len, k_len]`` on the host."""
    out = torch.zeros((batch, q_len, k_len), dtype=torch.bool)
    listed = lambda x, b: int(x[b]) if isinstance(x, (list, tuple, torch.Tensor)) else int(x)  # noqa: E731
    for b in range(batch):
        held = min(max(k_len if kv_len is None else listed(kv_len, b), 0), k_len)
        borders = [0, held]
        if lengths is not None:
            borders = [0, listed(lengths, b)]
        if documents is not None:
            rows = torch.as_tensor(documents).tolist()
            borders = rows[b] if isinstance(rows[0], list) else rows
        for i in range(q_len):
            t = held - q_len + i
            home = [(x, min(y, held)) for x, y in zip(borders, borders[1:]) if x <= t < y] if t >= 0 else []
            if not home:
                continue
            x, y = home[0]
            for j in range(max(x, 0), y):
                reached = not causal or (j - x) // chunk <= (t - x) // chunk
                near = window is None or (j > t - window and (causal or j < t + window))
                out[b, i, j] = (reached and (near or j - x < sink)) or j - x < listed(prefix, b)
    return out


def of_runs(given, k_len):
    """bool ``[B, Lq, k_len]`` of rows' runs."""
    j = torch.arange(k_len)
    r = given.cpu().long()[..., None]
    return ((j >= r[:, :, 0]) & (j < r[:, :, 1])) | ((j >= r[:, :, 2]) & (j < r[:, :, 3]))


def attention(q, k, v, mask, *, scale=None, cap=None, slopes=None, kv_len=None):
    """``(out [B, Lq, H, D], lse [B, H, Lq], parts)`` in fp64; ``parts``: the weights, the derivative of the cap and the distances.
    A row that sees nothing gets 0 and -inf. ``mask``: bool ``[B or 1, Lq, Lk]``."""
    b, n, h, d = q.shape
    m, hk = k.shape[1:3]
    mask = mask.to(q.device).expand(b, n, m)[:, None]
    scale = d ** -0.5 if scale is None else scale
    qh, kh, vh = (x.double().transpose(1, 2) for x in (q, k, v))
    kh, vh = (x.repeat_interleave(h // hk, dim=1) for x in (kh, vh))
    x = torch.matmul(qh, kh.transpose(-1, -2).contiguous()) * scale
    turn = torch.ones_like(x)
    if cap:
        bent = torch.tanh(x / cap)
        x, turn = cap * bent, 1 - bent ** 2
    held = torch.as_tensor(m if kv_len is None else kv_len).reshape(-1).expand(b).to(q.device).clamp(0, m)
    t = held[:, None] - n + torch.arange(n, device=q.device)
    far = (t[:, :, None] - torch.arange(m, device=q.device)).abs().double()[:, None]
    if slopes is not None:
        x = x - slopes.double()[:, None, None] * far
    any_seen = mask.any(-1, keepdim=True)
    x = torch.where(mask, x, -math.inf)
    lse = torch.logsumexp(torch.where(any_seen, x, 0.0), -1, keepdim=True)
    p = torch.where(mask, (x - lse).exp(), 0.0)
    out = torch.matmul(p, vh).transpose(1, 2)
    lse = torch.where(any_seen, lse, -math.inf)[..., 0]
    return out, lse, (p, turn, far)
