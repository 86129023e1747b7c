"""Attention of single queries over key blocks that a score selects from a KV cache (no reference
counterpart).

The framework's sparse branch routes whole blocks of queries (:mod:`.routing`); a token-by-token model
asks per token. :func:`select_key_blocks` scores the cache's key block sums, which
:func:`~worldattention_amd.hsa.kvcache.kv_append` keeps beside the keys, and chooses blocks for each
query and key head; :func:`selected_attention` attends to the chosen blocks; :func:`attend_selected`
does both on a ``kv_cache`` dict. They serve a decoding step, a few drafted tokens or a chunk of a prompt.
There is no gradient: training at this granularity runs
:func:`~worldattention_amd.hsa.block_sparse.block_sparse_attention` from a block map.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Union

import torch

from .. import _lib

__all__ = ["BlockSelection", "select_key_blocks", "selected_attention", "attend_selected"]


class BlockSelection(NamedTuple):
    """Chosen key blocks of each query: ``index`` int32 ``[B, n, Hk, topk]``, ascending, -1 behind the
    first ``num`` int32 ``[B, n, Hk]``."""

    index: torch.Tensor
    num: torch.Tensor


KvLen = Union[int, torch.Tensor]


def _check_query(q, kv_heads: int, bsz: int, d: int, block_size: int, kv_len: KvLen) -> None:
    if q.dim() != 4 or q.shape[0] != bsz or q.shape[3] != d:
        raise ValueError(f"q must be [B={bsz}, n, H, D={d}], got {tuple(q.shape)}")
    heads = q.shape[2]
    if d not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {d}")
    if kv_heads < 1 or heads % kv_heads or heads < kv_heads:
        raise ValueError(f"{heads} query heads do not share {kv_heads} key heads")
    if block_size not in (64, 128):
        raise ValueError(f"block_size must be 64 or 128, got {block_size}")
    if q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bf16, got {q.dtype}")
    if isinstance(kv_len, torch.Tensor) and (tuple(kv_len.shape) != (bsz,) or kv_len.dtype != torch.int32):
        raise ValueError(f"kv_len must be an int or int32 [{bsz}], got {kv_len.dtype} {tuple(kv_len.shape)}")


def _no_gradient(*tensors) -> None:
    _lib.refuse_tangents(*tensors)
    if not torch.is_grad_enabled():
        return
    for t in tensors:
        if not t.requires_grad:
            continue
        raise ValueError("attention over selected cache blocks takes no gradient: call it under torch.no_grad(), or train "
                         "with block_sparse_attention(block_map=...)")


def _lengths(kv_len: KvLen):
    """``(tensor or None, pointer, value)``."""
    if isinstance(kv_len, torch.Tensor):
        kv_len = kv_len.contiguous()
        return kv_len, kv_len.data_ptr(), 0
    return None, None, int(kv_len)


def _select(q, sums, kv_len, bs, topk, sink, local, cap) -> BlockSelection:
    dev = q.device
    bsz, n, heads, d = q.shape
    hk, nb = sums.shape[1:3]
    index = torch.empty(bsz, n, hk, topk, dtype=torch.int32, device=dev)
    num = torch.empty(bsz, n, hk, dtype=torch.int32, device=dev)
    if bsz == 0 or n == 0:
        return BlockSelection(index, num)
    size = _lib.sizes("wa_select_blocks_workspace_bytes", bsz, n, hk, nb)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    keep, len_ptr, len_all = _lengths(kv_len)
    args = _lib.SelectBlocksArgs(*_lib.blhd(q), sums.data_ptr(), nb, len_ptr, len_all, cap, bsz, n, heads, hk, d, bs, topk,
                                 sink, local, index.data_ptr(), num.data_ptr(), _lib.ptr(ws))
    _lib.launch("wa_select_blocks", args, dev)
    return BlockSelection(index, num)


def _attend(q, k, v, index, num, kv_len, bs, scale):
    dev = q.device
    bsz, n, heads, d = q.shape
    cap, hk = k.shape[1:3]
    out = torch.empty(bsz, n, heads, d, dtype=torch.bfloat16, device=dev)
    lse = torch.empty(bsz, heads, n, dtype=torch.float32, device=dev)
    if bsz == 0 or n == 0:
        return out, lse
    topk = index.shape[-1]
    size = _lib.sizes("wa_selected_attn_workspace_bytes", bsz, n, heads, hk, d, topk, bs)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    keep, len_ptr, len_all = _lengths(kv_len)
    args = _lib.SelectedAttnArgs(*_lib.blhd(q), *_lib.blhd(k), *_lib.blhd(v), *_lib.blhd(out), lse.data_ptr(),
                                 index.data_ptr(), num.data_ptr(), topk, len_ptr, len_all, bsz, n, cap, heads, hk, d, bs,
                                 scale, _lib.ptr(ws))
    _lib.launch("wa_selected_attn", args, dev)
    return out, lse


def _scale_arg(scale: Optional[float]) -> float:
    """The kernel's fp32 scale, whose 0 stands for the default."""
    if scale is None:
        return 0.0
    scale = float(scale)
    if ctypes.c_float(scale).value == 0.0:
        raise ValueError(f"scale must not be 0 in fp32, got {scale}")
    return scale


def _check_budget(topk: int, sink: int, local: int) -> None:
    if sink < 0 or local < 1 or sink + local > topk or topk > _lib.SELECT_MAX_BLOCKS:
        raise ValueError(f"topk {topk} (at most {_lib.SELECT_MAX_BLOCKS}) must hold {sink} sink and {local} (at least 1) local "
                         "blocks")


def _check_sums(sums, what: str) -> None:
    if sums.dim() != 4 or sums.dtype is not torch.float32 or not sums.is_contiguous():
        raise ValueError(f"{what} must be contiguous fp32 [B, Hk, blocks, D], got {sums.dtype} {tuple(sums.shape)}")
    if not 1 <= sums.shape[2] <= _lib.SELECT_MAX_BLOCKS:
        raise ValueError(f"{what} must hold 1 to {_lib.SELECT_MAX_BLOCKS} blocks, got {sums.shape[2]}")


def _readable(strides) -> bool:
    sb, st, sh, sc = strides
    return sc == 1 and sb % 8 == 0 and st % 8 == 0 and sh % 8 == 0 and st <= 1 << 24


def _check_cache(k, v) -> None:
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"cache k / v must be matching [B, cap, Hk, D] tensors, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError(f"cache k / v must be bf16, got {k.dtype} and {v.dtype}")
    strides = k.stride()
    if (k.shape[1] < 1 or not _readable(strides) or (v.stride() != strides and not _readable(v.stride()))
            or k.data_ptr() % 16 or v.data_ptr() % 16):
        raise ValueError("cache k / v must hold tokens, with contiguous channels in 16-byte aligned rows at most 2^24 elements "
                         "apart (a cache is read in place)")


def select_key_blocks(q: torch.Tensor, k_block_sums: torch.Tensor, kv_len: KvLen, *, block_size: int, topk: int,
                      sink_blocks: int = 1, local_blocks: int = 1) -> BlockSelection:
    """Choose up to ``topk`` key blocks of a cache for each query and key head.

    * ``q``: bf16 ``[B, n, H, D]``, each sequence's last ``n`` tokens (their keys are in the cache already):
      query ``i`` sits at token ``kv_len[b] - n + i`` and sees the tokens up to its own.
    * ``k_block_sums``: fp32 ``[B, Hk, blocks, D]`` as ``kv_append`` keeps them; ``H`` is a multiple of ``Hk``,
      and the ``H / Hk`` query heads of a key head share its choice.
    * ``kv_len``: an int, or int32 ``[B]`` on the GPU (clamped to what the blocks hold).

    The first ``sink_blocks`` and last ``local_blocks`` (at least the query's own) seen blocks are always
    chosen, then the highest of ``(sum of the group's queries) . (sum of the block's keys)``, in fp64; ties
    go to the lowest block. (Scores closer than the rounding of such a sum, ``D 2^-52`` of its products' magnitudes,
    can rank differently for a single query and among several; equal key sums always tie.) A query before its
    sequence's first token gets none.
    """
    _check_sums(k_block_sums, "k_block_sums")
    bsz, hk, _, d = k_block_sums.shape
    _check_query(q, hk, bsz, d, block_size, kv_len)
    _check_budget(topk, sink_blocks, local_blocks)
    _no_gradient(q, k_block_sums)
    _lib.require_gpu(q, k_block_sums, kv_len if isinstance(kv_len, torch.Tensor) else None)
    return _select(_lib.kernel_ready(q), k_block_sums, kv_len, block_size, int(topk), int(sink_blocks), int(local_blocks), 0)


def selected_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, index: torch.Tensor, num: torch.Tensor,
                       kv_len: KvLen, *, block_size: int, scale: Optional[float] = None):
    """``(out [B, n, H, D] bf16, lse [B, H, n] fp32)`` of softmax attention over the first ``num`` listed blocks.

    ``q``, ``kv_len`` as in :func:`select_key_blocks`; ``k``, ``v``: bf16 cache ``[B, cap, Hk, D]``, read in place;
    ``index`` int32 ``[B, n, Hk, width]``, ``num`` int32 ``[B, n, Hk]``: any lists (an id without seen tokens adds
    nothing, a repeated one counts again). A query that sees nothing gets 0 and ``lse = -inf``; what the cache
    holds behind a sequence's end is not used. ``scale``: default ``D ** -0.5``.
    """
    _check_cache(k, v)
    bsz, _, hk, d = k.shape
    _check_query(q, hk, bsz, d, block_size, kv_len)
    if index.dim() != 4 or tuple(index.shape[:3]) != (bsz, q.shape[1], hk) or tuple(num.shape) != (bsz, q.shape[1], hk):
        raise ValueError(f"index / num must be [{bsz}, {q.shape[1]}, {hk}, width] and [{bsz}, {q.shape[1]}, {hk}], got "
                         f"{tuple(index.shape)} and {tuple(num.shape)}")
    if index.dtype != torch.int32 or num.dtype != torch.int32 or not 1 <= index.shape[3] <= _lib.SELECT_MAX_BLOCKS:
        raise ValueError(f"index / num must be int32 with 1 to {_lib.SELECT_MAX_BLOCKS} ids a row, got {index.dtype}, {num.dtype} "
                         f"and {index.shape[3]}")
    scale = _scale_arg(scale)
    _no_gradient(q, k, v)
    _lib.require_gpu(q, k, v, index, num, kv_len if isinstance(kv_len, torch.Tensor) else None)
    return _attend(_lib.kernel_ready(q), k, v, index.contiguous(), num.contiguous(), kv_len, block_size, scale)


def attend_selected(q: torch.Tensor, kv_cache: dict, kv_len: KvLen, *, topk: int, sink_blocks: int = 1,
                    local_blocks: int = 1, scale: Optional[float] = None):
    """``(out, lse, BlockSelection)``: :func:`select_key_blocks` and :func:`selected_attention` on a cache that
    ``kv_append`` or ``cache_step`` keeps with a ``block_size`` (``kv_cache["k"]``, ``["v"]``, ``["k_block_sums"]``)."""
    if "k_block_sums" not in kv_cache or "k_block_sums_block_size" not in kv_cache:
        raise ValueError("kv_cache keeps no k_block_sums: write it with kv_append(..., block_size=...)")
    k, v, sums = kv_cache["k"], kv_cache["v"], kv_cache["k_block_sums"]
    bs = int(kv_cache["k_block_sums_block_size"])
    _check_cache(k, v)
    bsz, cap, hk, d = k.shape
    _check_query(q, hk, bsz, d, bs, kv_len)
    _check_sums(sums, "k_block_sums")
    if sums.shape != (bsz, hk, -(-cap // bs), d):
        raise ValueError(f"k_block_sums must be [{bsz}, {hk}, {-(-cap // bs)}, {d}], got {tuple(sums.shape)}")
    _check_budget(topk, sink_blocks, local_blocks)
    scale = _scale_arg(scale)
    _no_gradient(q, k, v, sums)
    _lib.require_gpu(q, k, v, sums, kv_len if isinstance(kv_len, torch.Tensor) else None)
    q = _lib.kernel_ready(q)
    chosen = _select(q, sums, kv_len, bs, int(topk), int(sink_blocks), int(local_blocks), cap)
    out, lse = _attend(q, k, v, chosen.index, chosen.num, kv_len, bs, scale)
    return out, lse, chosen
