"""Causal linear attention with a decay for each head (no reference counterpart).

The framework's linear heads (elu(x) + 1, ``wa_elu1_*``) read a whole window at once. These carry a
state from token to token instead, ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T`` and
``o_t = scale q_t S_t``: :func:`decay_linear_attention` for prompts and training (parallel over
segments of the sequence), :func:`decay_linear_step` for single tokens, on the same state.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .block_sparse import padded_head_dim

__all__ = ["decay_linear_attention", "decay_linear_step"]


def _ready(t: torch.Tensor) -> torch.Tensor:
    """``t`` in rows that the kernels take: 16-byte aligned, tokens at most 2^23 elements apart and, in bf16 (whose kernels
    cut rows off by a byte range), each behind the one before it: expanded and overlapping tokens are copied."""
    shared = t.dtype is torch.bfloat16 and t.shape[1] > 1 and t.stride(1) < t.shape[3]
    if shared or t.stride(1) > 1 << 23:
        t = t.clone(memory_format=torch.contiguous_format)   # contiguous() leaves a single token's stride as it is
    return _lib.kernel_ready(t, t.dtype, 16 // t.element_size())


def _forward(q, k, v, log_decay, initial, lengths, scale, want_derivs=False):
    dev = q.device
    bsz, length, heads, d = q.shape
    f32 = dict(dtype=torch.float32, device=dev)
    out = torch.empty((bsz, length, heads, d), dtype=q.dtype, device=dev)
    if out.numel() == 0:      # no tokens: the state passes through
        final = torch.zeros((bsz, heads, d, d), **f32) if initial is None else initial.clone()
        return out, final, None, None
    final = torch.empty((bsz, heads, d, d), **f32)
    n_seg = _lib.sizes("wa_decay_segments", bsz, length, heads, int(want_derivs))
    states = torch.empty((bsz, heads, n_seg, d, d), **f32)
    derivs = torch.empty((bsz, heads, n_seg + 1, d, d), **f32) if want_derivs else None
    args = _lib.DecayFwdArgs(*_lib.blhd(q), *_lib.blhd(k), *_lib.blhd(v), *_lib.blhd(out), _lib.dtype_code(q), bsz, length,
                             heads, d, log_decay.data_ptr(), _lib.ptr(lengths), _lib.ptr(initial), final.data_ptr(),
                             states.data_ptr(), _lib.ptr(derivs), scale)
    _lib.launch("wa_decay_fwd", args, dev)
    return out, final, states, derivs


class _DecayLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, lengths, scale):
        ctx.set_materialize_grads(False)
        out, final, states, derivs = _forward(q, k, v, log_decay, initial, lengths, scale, ctx.needs_input_grad[3])
        ctx.save_for_backward(q, k, v, log_decay, lengths, states, derivs)
        ctx.scale = scale
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, log_decay, lengths, states, derivs = ctx.saved_tensors
        if dout is None and dfinal is None:
            return None, None, None, None, None, None, None
        dev = q.device
        bsz, length, heads, d = q.shape
        f32 = dict(dtype=torch.float32, device=dev)
        if q.numel() == 0:
            dlog = torch.zeros((heads,), **f32) if ctx.needs_input_grad[3] else None
            dinitial = None
            if ctx.needs_input_grad[4]:
                dinitial = torch.zeros((bsz, heads, d, d), **f32) if dfinal is None else dfinal.clone()
            return *(torch.zeros_like(t) for t in (q, k, v)), dlog, dinitial, None, None
        dout = torch.zeros_like(q, memory_format=torch.contiguous_format) if dout is None else _ready(dout)
        dfinal = None if dfinal is None else dfinal.contiguous()
        dq, dk, dv = (torch.empty((bsz, length, heads, d), dtype=q.dtype, device=dev) for _ in range(3))
        dinitial = torch.empty((bsz, heads, d, d), **f32) if ctx.needs_input_grad[4] else None
        dlog = torch.empty((heads,), **f32) if ctx.needs_input_grad[3] else None
        size = _lib.sizes("wa_decay_bwd_workspace_bytes", bsz, length, heads, d, int(derivs is not None))
        ws = torch.empty((size,), dtype=torch.uint8, device=dev)
        args = _lib.DecayBwdArgs(*_lib.blhd(q), *_lib.blhd(k), *_lib.blhd(v), *_lib.blhd(dout), *_lib.blhd(dq),
                                 *_lib.blhd(dk), *_lib.blhd(dv), _lib.dtype_code(q), bsz, length, heads, d,
                                 log_decay.data_ptr(), _lib.ptr(lengths), states.data_ptr(), _lib.ptr(derivs), _lib.ptr(dfinal),
                                 _lib.ptr(dinitial), _lib.ptr(dlog), ws.data_ptr(), ctx.scale)
        _lib.launch("wa_decay_bwd", args, dev)
        return dq, dk, dv, dlog, dinitial, None, None


def _check(q, k, v, log_decay, state, what):
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or (v.shape != q.shape and v.shape[:3] != q.shape[:3]):
        raise ValueError(f"q and k must be [B, L, H, D] and v [B, L, H, Dv], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError(f"q, k and v must have one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    bsz, _, heads, d = q.shape
    if log_decay.shape != (heads,) or log_decay.dtype is not torch.float32:
        raise ValueError(f"log_decay must be fp32 [{heads}], got {log_decay.dtype} {tuple(log_decay.shape)}")
    shape = (bsz, heads, d, v.shape[-1])
    if state is not None and (state.shape != shape or state.dtype is not torch.float32):
        raise ValueError(f"{what} must be fp32 {shape}, got {state.dtype} {tuple(state.shape)}")


def decay_linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                           initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                           scale: Optional[float] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Outputs ``[B, L, H, Dv]`` and final state ``[B, H, D, Dv]`` (fp32) of the recurrence over whole sequences.

    * ``q``, ``k`` ``[B, L, H, D]`` and ``v`` ``[B, L, H, Dv]``: bf16 or fp32, any strides (a head dim shared by
      expansion included), head dims up to 128 (other than 64 and 128 they run zero-padded).
    * ``log_decay``: fp32 ``[H]``, not above 0 (``-inf``: the head sees its own token only).
    * ``initial_state``: fp32 ``[B, H, D, Dv]``, the state before the first token (default 0).
    * ``lengths``: int32 ``[B]`` on the GPU: sequence ``b`` is its first ``lengths[b]`` tokens (clamped to
      ``[0, L]``); the tokens behind are not read, their outputs and gradients are 0.
    * ``scale``: default ``D ** -0.5``; of any size, 0 too (the outputs are 0 then, the state is carried on).

    At most 65,535 sequences times heads. Outputs have the inputs' dtype; the state is summed in fp32. Differentiable
    once, through both results, in ``q``, ``k``, ``v``, ``log_decay`` and ``initial_state``. A value that is not finite in
    ``v`` (or, backwards, in the gradient) reaches its 64-token neighbourhood, as it reaches a tile of softmax
    attention. To capture a backward pass in a graph, capture its forward pass too, and let no eager graph of the same
    leaves live then.
    """
    _check(q, k, v, log_decay, initial_state, "initial_state")
    bsz, length, heads, d = q.shape
    dv = v.shape[-1]
    dp = padded_head_dim(max(d, dv))
    if lengths is not None and (tuple(lengths.shape) != (bsz,) or lengths.dtype != torch.int32):
        raise ValueError(f"lengths must be int32 [{bsz}], got {lengths.dtype} {tuple(lengths.shape)}")
    _lib.refuse_tangents(q, k, v, log_decay, initial_state)
    dev = _lib.require_gpu(q, k, v, log_decay, initial_state, lengths)
    _lib.dtype_code(q)
    scale = max(d, 1) ** -0.5 if scale is None else float(scale)
    if d != dp:
        q, k = (torch.nn.functional.pad(t, (0, dp - d)) for t in (q, k))
    if dv != dp:
        v = torch.nn.functional.pad(v, (0, dp - dv))
    if initial_state is not None:
        if d != dp or dv != dp:
            initial_state = torch.nn.functional.pad(initial_state, (0, dp - dv, 0, dp - d))
        initial_state = initial_state.contiguous()
    q, k, v = _ready(q), _ready(k), _ready(v)
    log_decay = log_decay.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, initial_state))
    if grad:
        out, final = _DecayLinear.apply(q, k, v, log_decay, initial_state, lengths, scale)
    else:
        out, final = _forward(q, k, v, log_decay, initial_state, lengths, scale)[:2]
    if d != dp or dv != dp:
        out, final = out[..., :dv].contiguous(), final[:, :, :d, :dv].contiguous()
    return out, final


def _apart(n: int, sn: int, m: int, sm: int, size: int) -> bool:
    """Whether ``n`` times ``m`` runs of ``size`` elements, strides ``sn`` and ``sm``, lie in memory of their own."""
    if (m == 1 or sm >= size) and (n == 1 or sn >= (m - 1) * sm + size):
        return True
    if (n == 1 or sn >= size) and (m == 1 or sm >= (n - 1) * sn + size):
        return True
    starts = sorted(i * sn + j * sm for i in range(n) for j in range(m))   # neither within the other: one by one
    return all(y - x >= size for x, y in zip(starts, starts[1:]))


def decay_linear_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *,
                      scale: Optional[float] = None) -> torch.Tensor:
    """The recurrence for single tokens: ``[B, L, H, D]`` with ``L`` 1 (or a few, one after the other), ``state``
    ``[B, H, D, Dv]`` fp32 updated in place (sequences and heads in memory of their own), outputs ``[B, L, H, Dv]``
    returned. Head dims up to 256, at most 65,535 sequences and as many heads. Not differentiable: inputs that ask for a gradient are refused while gradients
    are enabled."""
    _check(q, k, v, log_decay, state, "state")
    bsz, length, heads, d = q.shape
    dv = v.shape[-1]
    if d > 256 or dv > 256:
        raise ValueError(f"head dims must be at most 256, got {d} and {dv}")
    s_sb, s_sh, s_row, s_col = state.stride()
    if s_col != 1 or (d > 1 and s_row != dv):
        raise ValueError("the state's [D, Dv] matrices must be contiguous")
    if not _apart(bsz, s_sb, heads, s_sh, d * dv):
        raise ValueError("the state is updated in place: every sequence and head needs memory of its own")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                    or state.requires_grad):
        raise ValueError("decay_linear_step takes no gradient (decay_linear_attention does): call it under torch.no_grad()")
    _lib.refuse_tangents(q, k, v, log_decay, state)
    dev = _lib.require_gpu(q, k, v, log_decay, state)
    dtype = _lib.dtype_code(q)
    out = torch.empty(bsz, length, heads, dv, dtype=q.dtype, device=dev)
    if out.numel() == 0 or d == 0:
        return out.zero_()
    q, k, v = [t if t.stride(-1) == 1 else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v)]
    log_decay = log_decay.contiguous()
    args = _lib.DecayStepArgs(*_lib.blhd(q), *_lib.blhd(k), *_lib.blhd(v), *_lib.blhd(out), dtype, bsz, length, heads, d, dv,
                              log_decay.data_ptr(), state.data_ptr(), s_sb, s_sh, d ** -0.5 if scale is None else float(scale))
    _lib.launch("wa_decay_step", args, dev)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)   # a graph that saved the state must not use what it has become
    return out
