"""Rotary positions with several axes for token-by-token attention (no reference counterpart).

The cache step's RoPE (:func:`~worldattention_amd.hsa.kvcache.qkv_epilogue`) rotates a chunk on a
regular frame x height x width grid from a table. :func:`rope_axes` takes each token's position on
each axis, so video, image, text and action tokens mix in one sequence and lie as far out as an
integer reaches, and it is differentiable. :func:`axis_frequencies` gives the frequencies of the
framework's own 3-D table.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from .. import _lib

__all__ = ["axis_frequencies", "rope_axes"]


def axis_frequencies(head_dim: int, axes: int = 3, theta: float = 10000.0, device=None):
    """``(inv_freq, sections)`` of the model's axis split: with three axes the pairs of a head go to
    time, height and width as ``half - 2 * (half // 3)``, ``half // 3``, ``half // 3``
    (``wan/modules/causal_model.py:34-62``); fewer axes drop the last ones. Each axis has its own
    geometric run of frequencies ``theta ** -(i / pairs)``. ``inv_freq`` is fp64 ``[head_dim // 2]``."""
    if head_dim < 2 or axes not in (1, 2, 3):
        raise ValueError(f"head_dim must be at least 2 and axes 1, 2 or 3, got {head_dim} and {axes}")
    half = head_dim // 2
    third = half // 3
    sections = {1: (half,), 2: (half - third, third), 3: (half - 2 * third, third, third)}[axes]
    inv = [theta ** -(torch.arange(s, dtype=torch.float64) / max(s, 1)) for s in sections]
    return torch.cat(inv).to(device), sections


def _launch(q, k, positions, inv_freq, sections, interleaved, inverse):
    """Rotated copies of the tensors given (either may be None)."""
    q_src, q_out, q_fields, q_heads = _side(q)     # the sources are held until the launch: one may be a copy
    k_src, k_out, k_fields, k_heads = _side(k)
    some = q if q is not None else k
    bsz, length, _, d = some.shape
    places = positions.stride()
    args = _lib.RopeAxesArgs(*q_fields, *k_fields, _lib.dtype_code(some), bsz, length, q_heads, k_heads, d, positions.data_ptr(),
                             *(places if len(places) == 3 else (0, *places)), positions.dtype is torch.int64,
                             inv_freq.data_ptr(), len(sections), _lib.RopeSections(*sections), interleaved, inverse)
    _lib.launch("wa_rope_axes", args, positions.device)
    return q_out, k_out


def _side(t):
    """What the kernel reads for a tensor, its output, their argument fields and the heads."""
    if t is None:
        return None, None, (None, 0, 0, 0, None, 0, 0, 0), 0
    bsz, length, heads, d = t.shape
    out = torch.empty(bsz, length, heads, d, dtype=t.dtype, device=t.device)
    sb, st, sh, sc = t.stride()
    if sc != 1 and d != 1:
        t = t.contiguous()
        sb, st, sh, _ = t.stride()
    ob, ot, oh, _ = out.stride()
    return t, out, (t.data_ptr(), sb, st, sh, out.data_ptr(), ob, ot, oh), heads


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, sections, interleaved):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = sections, interleaved
        out, k_out = _launch(q, k, positions, inv_freq, sections, interleaved, False)
        return out if k is None else (out, k_out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        positions, inv_freq = ctx.saved_tensors
        if dq is None and dk is None:
            return None, None, None, None, None, None
        return (*_launch(dq, dk, positions, inv_freq, *ctx.how, True), None, None, None, None)


def rope_axes(q: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections: Sequence[int], *,
              k: Optional[torch.Tensor] = None, interleaved: bool = True):
    """Rotate ``q`` ``[B, L, H, D]`` (and ``k`` ``[B, L, Hk, D]``, in the same launch) to its tokens' positions.

    * ``positions``: int32 or int64 ``[L, axes]`` or ``[B, L, axes]``, any sign and size.
    * ``inv_freq``: ``[P]`` frequencies of the rotated pairs, fp64 (fp32 is converted), ``2 P <= D``;
      ``sections``: how many of them, in order, turn with each axis (up to four axes). Pair ``p`` turns by
      ``positions[..., axis(p)] * inv_freq[p]``. Channels from ``2 P`` on are copied.
    * ``interleaved``: pair ``p`` is channels ``(2p, 2p + 1)`` (the model's own layout); otherwise
      ``(p, p + P)``.

    bf16 or fp32; the angle's fraction of a revolution is exact to 2^-40 at any position (frequencies up to 1), the
    rotation is fp32, one rounding. Returns new contiguous tensors (``q``'s, or ``(q, k)``'s). Differentiable once in
    ``q`` and ``k``. To capture a backward pass in a graph, capture its forward pass too, and let no eager graph of
    the same leaves live then.
    """
    sections = tuple(map(int, sections))
    if q.dim() != 4:
        raise ValueError(f"q must be [B, L, H, D], got {tuple(q.shape)}")
    if k is not None and k.dim() != 4:
        raise ValueError(f"k must be [B, L, H, D], got {tuple(k.shape)}")
    bsz, length, _, d = q.shape
    if k is not None and (k.shape[0] != bsz or k.shape[1] != length or k.shape[3] != d or k.dtype != q.dtype):
        raise ValueError(f"k must hold q's tokens and head dim in its dtype, got {tuple(k.shape)} {k.dtype} for "
                         f"{tuple(q.shape)} {q.dtype}")
    axes, pairs = len(sections), sum(sections)
    if not 1 <= axes <= _lib.ROPE_MAX_AXES or min(sections) < 0 or pairs < 1:
        raise ValueError(f"sections must be 1 to {_lib.ROPE_MAX_AXES} pair counts, got {sections}")
    if d > _lib.ROPE_MAX_DIM or 2 * pairs > d:
        raise ValueError(f"{pairs} pairs do not fit a head dim of {d} (at most {_lib.ROPE_MAX_DIM})")
    if positions.shape != (bsz, length, axes) and positions.shape != (length, axes):
        raise ValueError(f"positions must be [{length}, {axes}] or [{bsz}, {length}, {axes}], got "
                         f"{tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if inv_freq.shape != (pairs,) or inv_freq.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"inv_freq must be [{pairs}] in fp64 or fp32, got {tuple(inv_freq.shape)} {inv_freq.dtype}")
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise ValueError("inv_freq takes no gradient: detach it")
    _lib.refuse_tangents(q, k, inv_freq)
    _lib.require_gpu(q, k, positions, inv_freq)
    _lib.dtype_code(q)
    inv_freq = inv_freq.double().contiguous()
    interleaved = bool(interleaved)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _RopeAxes.apply(q, k, positions, inv_freq, sections, interleaved)
    out, k_out = _launch(q, k, positions, inv_freq, sections, interleaved, False)
    return out if k is None else (out, k_out)
