"""Plain 64-bit forms of the 8-bit cache: codes and scales token block by token block, and attention over the values that they stand
for. Written from the definitions; on the host."""
from __future__ import annotations

import math

import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def nearest(x, dtype):
    """fp64 ``x`` to the nearest value that a code has, ties to the even code."""
    if dtype is torch.int8:
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)   # three bits behind the first, or 2^-9
    return torch.round(x / step) * step


def scale_for(largest: float, dtype) -> float:
    if not math.isfinite(largest):
        return math.nan
    e = -126
    while largest > LARGEST[dtype] * 2.0 ** e:
        e += 1
    return 2.0 ** e


class Cache:
    """One tensor (keys or values) of a cache: codes as fp64 numbers ``[B, cap, Hk, D]`` and scales ``[B, Hk, blocks]``."""

    def __init__(self, codes, scale, block_size, dtype):
        self.codes, self.scale, self.bs, self.dtype = codes.double().cpu(), scale.double().cpu(), block_size, dtype

    def append(self, new, starts, counts):
        """Also the touched blocks' sums of values: ``{(b, head, block): [D]}``."""
        sums = {}
        new = new.double().cpu()
        cap = self.codes.shape[1]
        for b, (start, count) in enumerate(zip(starts, counts)):
            count = min(max(count, 0), new.shape[1])
            if start < 0 or start + count > cap or count == 0:
                continue
            for block in range(start // self.bs, (start + count - 1) // self.bs + 1):
                lo, hi = block * self.bs, min((block + 1) * self.bs, start + count)
                first = max(lo, start)
                for h in range(new.shape[2]):
                    fresh = new[b, first - start: hi - start, h]
                    need = scale_for(float(fresh.abs().max()) if torch.isfinite(fresh).all() else math.nan, self.dtype)
                    old = float(self.scale[b, h, block]) if first > lo else 0.0
                    now = math.nan if math.isnan(need) or math.isnan(old) else max(need, old)
                    if not math.isnan(now):
                        if first > lo:
                            self.codes[b, lo:first, h] = nearest(self.codes[b, lo:first, h] * (old / now), self.dtype)
                        self.codes[b, first:hi, h] = nearest(fresh / now, self.dtype)
                    else:
                        self.codes[b, first:hi, h] = 0.0
                    self.scale[b, h, block] = now
                    sums[b, h, block] = self.codes[b, lo:hi, h].sum(0) * now
        return sums

    def values(self):
        cap = self.codes.shape[1]
        return self.codes * self.scale.repeat_interleave(self.bs, dim=2)[:, :, :cap].transpose(1, 2)[..., None]


def attend(q, k, v, kv_len, *, scale=None, cap=None, slopes=None, window=None, sink=0, chosen=None, block_size=64):
    """``(out [B, n, H, D], lse [B, H, n])`` of the newest tokens over values ``k``, ``v`` ``[B, cap, Hk, D]``. Ids listed twice count twice."""
    b, n, h, d = q.shape
    hk = k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    out, lse = torch.zeros((b, n, h, d), dtype=torch.float64), torch.full((b, h, n), -math.inf, dtype=torch.float64)
    for bi in range(b):
        held = min(max(int(kv_len[bi]), 0), k.shape[1])
        for i in range(n):
            t = held - n + i
            for hi in range(hk):
                if chosen is not None:
                    ids = chosen[0][bi, i, hi, :max(0, int(chosen[1][bi, i, hi]))].tolist()
                    at = [j for x in ids if x >= 0 for j in range(x * block_size, min(t + 1, (x + 1) * block_size))]
                else:
                    at = [j for j in range(t + 1) if not window or j > t - window or j < sink]
                if not at:
                    continue
                at = torch.tensor(at)
                for g in range(hi * (h // hk), (hi + 1) * (h // hk)):
                    s = scale * k[bi, at, hi] @ q[bi, i, g]
                    if cap:
                        s = cap * torch.tanh(s / cap)
                    if slopes is not None:
                        s = s - float(slopes[g]) * (t - at)
                    lse[bi, g, i] = torch.logsumexp(s, 0)
                    out[bi, i, g] = torch.softmax(s, 0) @ v[bi, at, hi]
    return out, lse
