"""Attention whose rows see ranges of keys, with capped scores and a bias by distance (no reference
counterpart).

The framework's sparse branch attends to whole blocks; a layer that trains on packed documents, on frames
that see themselves and those before them, or with a seen prefix, and a prompt under a window with sinks,
need masks by token. :func:`key_ranges` turns such rules into up to two runs of keys for each row, once for
a batch; :func:`ranged_attention` attends to them, forward and backward, in every layer.
:func:`~worldattention_amd.hsa.cache8.attend_8bit` is the same rule for single tokens over an 8-bit cache.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Union

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .block_sparse import padded_head_dim

__all__ = ["KeyRanges", "key_ranges", "ranged_attention"]

_MOST = 1 << 30      # tokens of a sequence
_FAR = 1 << 62       # of a whole number, which the kernels take in 64 bits


class KeyRanges(NamedTuple):
    """What the rows of a batch see: made by :func:`key_ranges`, read by :func:`ranged_attention`."""

    rows: torch.Tensor                    # int32 [B or 1, Lq, 4]: two disjoint runs of keys, the lower one second
    tiles: torch.Tensor                   # int32 [B or 1, ceil(Lq / 64), 12]: what 64 rows see together
    order: torch.Tensor                   # int32 [B or 1, ceil(Lq / 128) + ceil(Lk / 128) + 1]: tiles of rows and of keys, most work
                                          # first, and the first row's position
    q_len: int
    k_len: int


def _is_whole(x) -> bool:
    try:
        return not isinstance(x, bool) and int(x) == x
    except (OverflowError, ValueError):      # infinities and NaN
        return False


def _count(x, name: str, low: int) -> int:
    if not _is_whole(x) or not low <= x <= _FAR:
        raise ValueError(f"{name} must be a whole number of at least {low}, got {x}")
    return int(x)


def _per_sequence(x, bsz: int, name: str):
    """``(tensor or None, value)`` of an int or an int32 ``[B]``."""
    if isinstance(x, torch.Tensor):
        if tuple(x.shape) != (bsz,) or x.dtype is not torch.int32:
            raise ValueError(f"{name} must be an int or int32 [{bsz}], got {x.dtype} {tuple(x.shape)}")
        return x.contiguous(), 0
    if not _is_whole(x):
        raise ValueError(f"{name} must be a whole number or int32 [{bsz}], got {x}")
    if abs(x) > _FAR:
        raise ValueError(f"{name} does not fit 64 bits: {x}")
    return None, int(x)


def key_ranges(batch: int, q_len: int, k_len: int, *, causal: bool = True, chunk: int = 1, window: Optional[int] = None,
               sink: int = 0, prefix: Union[int, torch.Tensor] = 0, documents: Optional[torch.Tensor] = None,
               lengths: Optional[torch.Tensor] = None, kv_len: Union[int, torch.Tensor, None] = None,
               given: Optional[torch.Tensor] = None, device=None) -> KeyRanges:
    """The keys that each of ``q_len`` rows sees among ``k_len``, for ``batch`` sequences.

    Row ``i`` sits at key position ``t = kv_len - q_len + i`` (``kv_len``: int or int32 ``[B]`` on the GPU, default
    ``k_len``; a row before position 0 sees nothing) and, inside its document, sees

    * the keys up to its own; with ``chunk`` > 1 up to the end of its chunk of that many tokens, counted from the
      document's start (the frames of a video); all of them with ``causal=False``;
    * with ``window``, of the keys before its own only those less than ``window`` tokens back (with ``causal=False`` of those ahead too; a
      chunk's keys ahead are seen whatever the window), and still the document's first ``sink`` tokens (as far as the rules above
      reach);
    * the document's first ``prefix`` tokens (int, or int32 ``[B]``) from wherever it sits.

    ``documents``: int32 borders on the GPU, ascending, ``[n]`` for all sequences or ``[B, n]`` (repeat the last border
    to fill up a row): document ``d`` is ``[border d, border d + 1)``, and tokens outside all of them are padding that sees
    nothing and that nothing sees (a document that begins before token 0 keeps its count from there). ``lengths``: int32 ``[B]``, for a
    padded batch: one document of that many tokens. Without either a sequence is one document. Keys from ``kv_len`` on are seen by no row.

    ``given``: int32 ``[B or 1, q_len, 4]`` in place of all rules: rows' runs ``[0, 1)`` and ``[2, 3)`` (clamped to the keys; a
    key in both counts once; positions are used by a bias alone). A batch whose rules do not differ shares one set. Nothing is
    read back to the host, so ranges can be made, and captured, with device lengths.
    """
    return _make_ranges(batch, q_len, k_len, causal, chunk, window, sink, prefix, documents, lengths, kv_len, given, device)


def _make_ranges(batch, q_len, k_len, causal=True, chunk=1, window=None, sink=0, prefix=0, documents=None, lengths=None, kv_len=None,
                 given=None, device=None, in_order=False) -> KeyRanges:
    batch, q_len, k_len = _count(batch, "batch", 0), _count(q_len, "q_len", 0), _count(k_len, "k_len", 0)
    if q_len > _MOST or k_len > _MOST:
        raise ValueError(f"at most {_MOST} tokens, got {q_len} and {k_len}")
    chunk, sink = _count(chunk, "chunk", 1), _count(sink, "sink", 0)
    window = 0 if window is None else _count(window, "window", 1)
    if chunk > 1 and not causal:
        raise ValueError("chunk needs causal=True (without it a row sees its whole document)")
    if not isinstance(prefix, torch.Tensor):
        _count(prefix, "prefix", 0)
    if documents is not None and lengths is not None:
        raise ValueError("give documents or lengths: a padded batch's documents hold its lengths")
    prefix_t, prefix_all = _per_sequence(prefix, batch, "prefix")
    kv_len = k_len if kv_len is None else kv_len
    kv_t, kv_all = _per_sequence(kv_len, batch, "kv_len")
    if lengths is not None:
        if tuple(lengths.shape) != (batch,) or lengths.dtype is not torch.int32:
            raise ValueError(f"lengths must be int32 [{batch}], got {lengths.dtype} {tuple(lengths.shape)}")
        documents = torch.stack((torch.zeros_like(lengths), lengths), dim=1)
    docs_sb = n_borders = 0
    if documents is not None:
        if (documents.dtype is not torch.int32 or documents.dim() not in (1, 2) or documents.shape[-1] < 2
                or (documents.dim() == 2 and documents.shape[0] != batch)):
            raise ValueError(f"documents must be int32 borders [n >= 2] or [{batch}, n >= 2], got {documents.dtype} "
                             f"{tuple(documents.shape)}")
        documents = documents.contiguous()
        n_borders = documents.shape[-1]
        docs_sb = n_borders if documents.dim() == 2 else 0
    sets = batch
    if given is not None:
        if given.dim() != 3 or given.shape[0] not in (1, batch) or tuple(given.shape[1:]) != (q_len, 4) or given.dtype is not torch.int32:
            raise ValueError(f"given must be int32 [{batch} or 1, {q_len}, 4], got {given.dtype} {tuple(given.shape)}")
        sets = given.shape[0] if kv_t is None else batch
        given = given.expand(sets, q_len, 4).contiguous()
    elif kv_t is None and prefix_t is None and docs_sb == 0:
        sets = min(1, batch)
    dev = _lib.require_gpu(given, documents, prefix_t, kv_t)
    if dev is None:
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise RuntimeError(f"worldattention_amd runs its HIP kernels on a ROCm GPU only; got device {dev}")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
    elif device is not None and torch.device(device).type != "cuda":
        raise ValueError(f"tensors on {dev}, device {device}")
    rows = torch.empty((sets, q_len, 4), dtype=torch.int32, device=dev)
    tiles = torch.empty((sets, -(-q_len // 64), 12), dtype=torch.int32, device=dev)
    order = torch.empty((sets, -(-q_len // 128) - (-k_len // 128) + 1), dtype=torch.int32, device=dev)
    if rows.numel():
        args = _lib.KeyRangesArgs(sets, q_len, k_len, _lib.ptr(kv_t), kv_all, _lib.ptr(given), int(bool(causal)), chunk, window,
                                  sink, _lib.ptr(prefix_t), prefix_all, _lib.ptr(documents), docs_sb, n_borders, rows.data_ptr(),
                                  tiles.data_ptr(), order.data_ptr(), int(in_order))
        _lib.launch("wa_key_ranges", args, dev)
    return KeyRanges(rows, tiles, order, q_len, k_len)


def _ready(t: torch.Tensor) -> torch.Tensor:
    """``t`` in rows that the kernels take: 16-byte aligned, tokens at most 2^23 elements apart."""
    if not 0 <= t.stride(1) <= 1 << 23:
        t = t.clone(memory_format=torch.contiguous_format)
    return _lib.kernel_ready(t)


def _range_args(ranges: KeyRanges):
    return ranges.rows.data_ptr(), ranges.tiles.data_ptr(), ranges.order.data_ptr(), int(ranges.rows.shape[0] > 1)


def _forward(q, k, v, slopes, ranges, scale, cap):
    dev = q.device
    bsz, n, heads, d = q.shape
    out = torch.empty((bsz, n, heads, d), dtype=q.dtype, device=dev)
    lse = torch.empty((bsz, heads, n), dtype=torch.float32, device=dev)
    if out.numel() == 0 or k.shape[1] == 0:
        return out.zero_(), lse.fill_(-math.inf)
    size = _lib.sizes("wa_ranged_fwd_workspace_bytes", bsz, heads, k.shape[2], n, k.shape[1], d)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    args = _lib.RangedFwdArgs(*_lib.blhd(q), *_lib.blhd(k), *_lib.blhd(v), *_lib.blhd(out), lse.data_ptr(), *_range_args(ranges),
                              _lib.ptr(slopes), bsz, heads, k.shape[2], n, k.shape[1], d, scale, cap, _lib.ptr(ws))
    _lib.launch("wa_ranged_fwd", args, dev)
    return out, lse


class _Ranged(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, ranges, scale, cap):
        ctx.set_materialize_grads(False)
        out, lse = _forward(q, k, v, slopes, ranges, scale, cap)
        ctx.save_for_backward(q, k, v, slopes, out, lse, *ranges[:3])
        ctx.rest = (ranges.q_len, ranges.k_len, scale, cap)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlse):
        none = (None,) * 3
        if dout is None and dlse is None:
            return None, None, None, None, *none
        q, k, v, slopes, out, lse, *ranges = ctx.saved_tensors
        q_len, k_len, scale, cap = ctx.rest
        ranges = KeyRanges(*ranges, q_len, k_len)
        dev = q.device
        bsz, n, heads, d = q.shape
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
        want_slopes = slopes is not None and ctx.needs_input_grad[3]
        dslopes = torch.empty((heads,), dtype=torch.float32, device=dev) if want_slopes else None
        if out.numel() == 0 or k.shape[1] == 0:
            return dq.zero_(), dk.zero_(), dv.zero_(), dslopes.zero_() if want_slopes else None, *none
        dout = torch.zeros_like(out) if dout is None else _ready(dout)
        dlse = None if dlse is None else dlse.contiguous()
        size = _lib.sizes("wa_ranged_bwd_workspace_bytes", bsz, heads, k.shape[2], n, k.shape[1], d)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        args = _lib.RangedBwdArgs(*_lib.blhd(q), *_lib.blhd(k), *_lib.blhd(v), *_lib.blhd(out), *_lib.blhd(dout), lse.data_ptr(),
                                  _lib.ptr(dlse), *_range_args(ranges), _lib.ptr(slopes), bsz, heads, k.shape[2], n, k.shape[1], d,
                                  scale, cap, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.ptr(dslopes), ws.data_ptr())
        _lib.launch("wa_ranged_bwd", args, dev)
        return dq, dk, dv, dslopes, *none


def check_scores(d: int, heads: int, scale, cap, slopes) -> tuple[float, float]:
    """The kernels' fp32 ``(scale, cap)``, the cap's 0 for none, of the score options that the operators share."""
    scale = max(d, 1) ** -0.5 if scale is None else float(scale)
    cap = 0.0 if cap is None else float(cap)
    as_f32 = ctypes.c_float(scale).value
    if not 0.0 < as_f32 < math.inf:
        raise ValueError(f"scale must be above 0 and finite in fp32, got {scale}")
    if not 0.0 <= cap <= 1e6 or (cap > 0.0 and not 1e-6 <= cap):
        raise ValueError(f"cap must be between 1e-6 and 1e6 (None or 0: no cap), got {cap}")
    if cap > 0.0 and scale > 1e30:
        raise ValueError(f"scale must be at most 1e30 with a cap, got {scale}")
    if slopes is not None and (tuple(slopes.shape) != (heads,) or slopes.dtype is not torch.float32):
        raise ValueError(f"slopes must be fp32 [{heads}], got {slopes.dtype} {tuple(slopes.shape)}")
    return scale, cap


def ranged_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ranges: KeyRanges, *, scale: Optional[float] = None,
                     cap: Optional[float] = None, slopes: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Softmax attention of ``q`` ``[B, Lq, H, D]`` over the keys that its rows' ``ranges`` hold, ``[B, Lq, H, D]``.

    * ``k``, ``v``: ``[B, Lk, Hk, D]``; ``H`` is a multiple of ``Hk``, and ``H / Hk`` neighbouring query heads share a key
      head. All bf16, any strides; head dims up to 128 (other than 64 and 128 they run zero-padded).
    * ``ranges``: :func:`key_ranges` of these lengths, for this batch or for one sequence that all share.
    * scores: ``scale q.k`` (default ``D ** -0.5``; above 0), then with ``cap`` (1e-6 to 1e6) ``cap tanh(score / cap)``, then with
      ``slopes`` (fp32 ``[H]``) less ``slopes[h]`` times the distance of the row's and the key's positions.
    * ``return_lse``: also the log-sum-exp of each row's scores, fp32 ``[B, H, Lq]``.

    A row that sees nothing gets 0 and a log-sum-exp of ``-inf``, and gradients of 0. Differentiable once in ``q``, ``k``, ``v`` and
    ``slopes``, through both results; the gradient of a shared key head is the sum over its query heads. Sums and softmax
    statistics are fp32; weights are rounded to bf16 once, for the product that they enter, scores' gradients to bf16 for the keys' and to
    16 bits for the queries' gradients (for the keys', weights times the cap's derivative below 2^-26
    are off by up to 2^-37).
    Sums run in a fixed order. Gradients are formed from the fp32 log-sum-exp, so they lose accuracy where scores pass 2^16 in
    magnitude. Keys and values that none of 128 neighbouring rows sees are not read for them; a value that is
    not finite reaches, besides the rows that see it, rows that share its tile of 128 rows by 64 keys. In the gradients so do a key, for the
    queries', and, for the keys' and values' of its tile of 64 rows by 128 keys, a query or an output's gradient (rows behind the last of 64 that
    sees anything are not read).
    """
    if q.dim() != 4 or k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] or v.shape != k.shape:
        raise ValueError(f"q must be [B, Lq, H, D] and k, v matching [B, Lk, Hk, D], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if q.dtype is not torch.bfloat16 or k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16:
        raise ValueError(f"q, k and v must be bf16, got {q.dtype}, {k.dtype}, {v.dtype}")
    bsz, n, heads, d = q.shape
    hk = k.shape[2]
    if hk < 1 or heads < hk or heads % hk:
        raise ValueError(f"{heads} query heads do not share {hk} key heads")
    if ranges.q_len != n or ranges.k_len != k.shape[1] or ranges.rows.shape[0] not in (1, bsz):
        raise ValueError(f"ranges of {ranges.rows.shape[0]} sequences, {ranges.q_len} rows and {ranges.k_len} keys do not fit "
                         f"{bsz}, {n} and {k.shape[1]}")
    sets = ranges.rows.shape[0]
    shapes = ((sets, n, 4), (sets, -(-n // 64), 12), (sets, -(-n // 128) - (-k.shape[1] // 128) + 1))
    if any(t.shape != s or t.dtype is not torch.int32 or not t.is_contiguous() for t, s in zip(ranges, shapes)):
        raise ValueError("ranges must be as key_ranges makes them")
    dp = padded_head_dim(d)
    scale, cap = check_scores(d, heads, scale, cap, slopes)
    _lib.refuse_tangents(q, k, v, slopes)
    _lib.require_gpu(q, k, v, slopes, *ranges[:3])
    if d != dp:
        q, k, v = (torch.nn.functional.pad(t, (0, dp - d)) for t in (q, k, v))
    q, k, v = _ready(q), _ready(k), _ready(v)
    slopes = None if slopes is None else slopes.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (slopes is not None and slopes.requires_grad)):
        out, lse = _Ranged.apply(q, k, v, slopes, ranges, scale, cap)
    else:
        out, lse = _forward(q, k, v, slopes, ranges, scale, cap)
    if d != dp:
        out = out[..., :d].contiguous()
    return (out, lse) if return_lse else out
