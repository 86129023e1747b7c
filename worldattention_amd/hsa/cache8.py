"""A KV cache in 8 bits and the attention of the newest tokens over it (no reference counterpart).

Half the bytes of the bf16 cache that :func:`~worldattention_amd.hsa.kvcache.kv_append` writes, for a model that
decodes token by token from long caches. :func:`new_cache_8bit` makes the ``kv_cache`` dict, :func:`kv_append_8bit`
quantises tokens as it writes them, :func:`kv_read_8bit` reads values back for the paths that take bf16, and
:func:`attend_8bit` attends to the codes themselves, with the score rules of
:func:`~worldattention_amd.hsa.ranged.ranged_attention`: for single tokens, a few drafted ones, or a chunk of a prompt,
over the whole cache, a window with sinks, or the blocks that
:func:`~worldattention_amd.hsa.selected.select_key_blocks` chooses from its key sums.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _lib
from .ranged import _count, _forward, _make_ranges, _per_sequence, check_scores
from .selected import BlockSelection, KvLen

__all__ = ["new_cache_8bit", "kv_append_8bit", "kv_read_8bit", "attend_8bit"]

_CODES = {torch.int8: _lib.WA_CODE_INT8, torch.float8_e4m3fn: _lib.WA_CODE_E4M3}

# Rows of a key head (queries times query heads) up to which attend_8bit reads codes, once for every 32 or 64 rows; above, the values are
# read back to bf16 once. 8 key heads of 128, codes against read back: 256 rows 96 and 110 us over 32,760 tokens, 30 and 50 over 4,096, 615 and
# 723 for 8 sequences of 32,000; 512 rows 176 and 121, 39 and 50, 1,065 and 777.
_FEW_ROWS = 256


def new_cache_8bit(batch: int, cap: int, kv_heads: int, head_dim: int, *, block_size: int = 64, dtype=torch.int8,
                   device="cuda") -> dict:
    """An empty ``kv_cache`` dict of 8-bit codes:

    * ``k``, ``v``: ``dtype`` (``torch.int8`` or ``torch.float8_e4m3fn``) ``[B, cap, Hk, D]``, ``D`` 64 or 128;
    * ``k_scale``, ``v_scale``: fp32 ``[B, Hk, blocks]``, one for each head and block of ``block_size`` (64 or 128) tokens; a
      token's value is its code times the scale. Scales are powers of two, so the values are exact in bf16;
    * ``k_block_sums`` fp32 ``[B, Hk, blocks, D]`` and ``k_block_sums_block_size``, as ``kv_append`` keeps them.
    """
    if dtype not in _CODES:
        raise ValueError(f"dtype must be torch.int8 or torch.float8_e4m3fn, got {dtype}")
    if head_dim not in (64, 128) or block_size not in (64, 128):
        raise ValueError(f"head_dim and block_size must be 64 or 128, got {head_dim} and {block_size}")
    batch, cap, kv_heads = _count(batch, "batch", 1), _count(cap, "cap", 1), _count(kv_heads, "kv_heads", 1)
    blocks = -(-cap // block_size)
    codes = lambda: torch.zeros((batch, cap, kv_heads, head_dim), dtype=torch.uint8, device=device).view(dtype)  # noqa: E731
    scales = lambda: torch.zeros((batch, kv_heads, blocks), dtype=torch.float32, device=device)  # noqa: E731
    return {"k": codes(), "v": codes(), "k_scale": scales(), "v_scale": scales(),
            "k_block_sums": torch.zeros((batch, kv_heads, blocks, head_dim), dtype=torch.float32, device=device),
            "k_block_sums_block_size": block_size}


def _no_gradient(*tensors) -> None:
    _lib.refuse_tangents(*tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("an 8-bit cache takes no gradient: call it under torch.no_grad(), or train with ranged_attention")


def _cache_args(c: dict):
    """``(wa_cache8, its tensors)``."""
    try:
        k, v, ks, vs, bs = c["k"], c["v"], c["k_scale"], c["v_scale"], c["k_block_sums_block_size"]
    except KeyError as e:
        raise ValueError(f"kv_cache has no {e.args[0]}: make it with new_cache_8bit") from None
    if k.dim() != 4 or v.shape != k.shape or k.dtype not in _CODES or v.dtype is not k.dtype:
        raise ValueError(f"cache k / v must be matching int8 or e4m3 [B, cap, Hk, D], got {k.dtype} {tuple(k.shape)} and {v.dtype} "
                         f"{tuple(v.shape)}")
    bsz, cap, hk, d = k.shape
    if d not in (64, 128) or bs not in (64, 128):
        raise ValueError(f"head_dim and block_size must be 64 or 128, got {d} and {bs}")
    if k.numel() == 0:
        raise ValueError(f"the cache holds no tokens: {tuple(k.shape)}")
    blocks = -(-cap // bs)
    if (ks.shape != (bsz, hk, blocks) or vs.shape != ks.shape or ks.dtype is not torch.float32 or vs.dtype is not torch.float32):
        raise ValueError(f"k_scale / v_scale must be fp32 [{bsz}, {hk}, {blocks}], got {ks.dtype} {tuple(ks.shape)} and {vs.dtype} "
                         f"{tuple(vs.shape)}")
    sums = c.get("k_block_sums")
    if sums is not None and (sums.shape != (bsz, hk, blocks, d) or sums.dtype is not torch.float32):
        raise ValueError(f"k_block_sums must be fp32 [{bsz}, {hk}, {blocks}, {d}], got {sums.dtype} {tuple(sums.shape)}")
    tensors = [k, v, ks, vs] if sums is None else [k, v, ks, vs, sums]
    if not all(t.is_contiguous() for t in tensors) or k.data_ptr() % 16 or v.data_ptr() % 16:
        raise ValueError("the cache's tensors must be contiguous, its codes on 16-byte addresses (they are read and written in place)")
    return _lib.Cache8(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), _lib.ptr(sums), bsz, cap, hk, d, bs,
                       _CODES[k.dtype]), tensors


def check_cache_8bit(kv_cache: dict) -> None:
    """Refuse a dict that is not as :func:`new_cache_8bit` makes it."""
    _cache_args(kv_cache)


def _start(x, bsz: int, name: str):
    """``(tensor or None, pointer, value)`` of an int or an int32 ``[B]`` on the GPU."""
    x, value = _per_sequence(x, bsz, name)
    return x, _lib.ptr(x), value


def kv_append_8bit(kv_cache: dict, k_new: torch.Tensor, v_new: torch.Tensor, write_start: Union[int, torch.Tensor], *,
                   lengths: Optional[torch.Tensor] = None) -> None:
    """Write ``k_new`` / ``v_new`` ``[B, n, Hk, D]`` (bf16 or fp32) as codes into cache tokens ``[write_start, write_start + n)``.

    ``write_start``: an int, or int32 ``[B]`` on the GPU, a place for each sequence; ``lengths``: int32 ``[B]``, how many of the
    ``n`` each brings (default all). A sequence whose tokens would not fit the cache is left as it is (with an int that is
    refused).

    A block's scale is the smallest power of two (2^-126 at least) at which its values fit the codes (127 in int8, 448 in
    e4m3), and codes are rounded to nearest even. A write that begins a block sets its scale anew; one behind earlier tokens of
    the block keeps their scale or, if it needs a larger one, rounds their codes again at that: an int8 token is off by less
    than one step of its block's scale in all. What the block held behind the written tokens is given up (rejected drafts are
    overwritten this way). ``k_block_sums`` of the touched blocks are those of the keys that the codes stand for. A value that
    is not finite makes its block's scale NaN, and so every token of the block, until the block is begun anew; finite ones of more than
    1.9 2^127 may be rounded up to 2^128, which reads as infinite. Not differentiable; in place, on the current stream, and fit for graph capture.
    """
    c, tensors = _cache_args(kv_cache)
    bsz, cap, hk, d = tensors[0].shape
    if (k_new.shape != v_new.shape or k_new.dim() != 4 or k_new.shape[0] != bsz or tuple(k_new.shape[2:]) != (hk, d)
            or k_new.dtype is not v_new.dtype):
        raise ValueError(f"new k / v must be matching [B={bsz}, n, Hk={hk}, D={d}], got {k_new.dtype} {tuple(k_new.shape)} and "
                         f"{v_new.dtype} {tuple(v_new.shape)}")
    n = k_new.shape[1]
    start, start_ptr, start_all = _start(write_start, bsz, "write_start")
    if n > cap or (start is None and (start_all < 0 or start_all + n > cap)):
        raise ValueError(f"{n} tokens from {start_all} on do not fit a cache of {cap}")
    if lengths is not None and (tuple(lengths.shape) != (bsz,) or lengths.dtype is not torch.int32):
        raise ValueError(f"lengths must be int32 [{bsz}], got {lengths.dtype} {tuple(lengths.shape)}")
    _no_gradient(k_new, v_new)
    dev = _lib.require_gpu(*tensors, k_new, v_new, start, lengths)
    dtype = _lib.dtype_code(k_new)
    if n == 0:
        return
    k_new, v_new = (_lib.kernel_ready(t, t.dtype, 16 // t.element_size()) for t in (k_new, v_new))
    lengths = None if lengths is None else lengths.contiguous()
    args = _lib.Kv8AppendArgs(c, *_lib.blhd(k_new), *_lib.blhd(v_new), dtype, n, start_ptr, start_all, _lib.ptr(lengths))
    _lib.launch("wa_kv8_append", args, dev)


def _read(c, dev, start_ptr, start_all, n, dtype, kv=(None, -1), last=0, window=0, sink=0):
    k, v = (torch.empty((c.B, n, c.Hk, c.D), dtype=dtype, device=dev) for _ in range(2))
    if n:
        args = _lib.Kv8ReadArgs(c, k.data_ptr(), v.data_ptr(), _lib.dtype_code(k), n, start_ptr, start_all, *kv, last, window, sink)
        _lib.launch("wa_kv8_read", args, dev)
    return k, v


def kv_read_8bit(kv_cache: dict, start: Union[int, torch.Tensor], n: int, *, dtype=torch.bfloat16):
    """``(k, v)`` ``[B, n, Hk, D]`` (bf16, exactly what the codes stand for, or fp32) of cache tokens ``[start, start + n)``; ``start``:
    an int, or int32 ``[B]`` on the GPU. Tokens outside the cache read as 0, tokens that were never written as whatever
    the codes hold (0 in a new cache)."""
    c, tensors = _cache_args(kv_cache)
    n = _count(n, "n", 0)
    keep, start_ptr, start_all = _start(start, c.B, "start")
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"dtype must be bf16 or fp32, got {dtype}")
    dev = _lib.require_gpu(*tensors, keep)
    return _read(c, dev, start_ptr, start_all, n, dtype)


def attend_8bit(q: torch.Tensor, kv_cache: dict, kv_len: KvLen, *, scale: Optional[float] = None, cap: Optional[float] = None,
                slopes: Optional[torch.Tensor] = None, window: Optional[int] = None, sink: int = 0,
                chosen: Optional[BlockSelection] = None):
    """``(out [B, n, H, D] bf16, lse [B, H, n] fp32)`` of each sequence's ``n`` newest tokens over its 8-bit cache.

    * ``q``: bf16 ``[B, n, H, D]``; their keys are in the cache already: query ``i`` sits at token ``kv_len[b] - n + i`` and sees
      the tokens up to its own (one before the first token sees nothing: 0 and ``-inf``). ``H`` is a multiple of ``Hk``.
    * ``kv_len``: an int, or int32 ``[B]`` on the GPU (clamped to the cache). What lies behind is not used.
    * ``scale``, ``cap``, ``slopes``: the scores', as in :func:`~worldattention_amd.hsa.ranged.ranged_attention`.
    * ``window``: only the ``window`` newest tokens, a query's own among them, and the first ``sink``.
    * ``chosen``: a :class:`~worldattention_amd.hsa.selected.BlockSelection` instead (no window): each query and key head attends
      to the seen tokens of its listed blocks (any lists; an id listed twice counts twice).

    Few queries (up to 256 rows, queries times heads, of a key head) and chosen blocks read the codes; a longer chunk reads the
    tokens that it sees back into bf16 once, exactly, and attends to those: two tensors of ``[B, cap, Hk, D]`` while the call
    runs. Sums and softmax statistics are fp32; weights (times the values' scale) round to bf16 once. No gradient.
    """
    c, tensors = _cache_args(kv_cache)
    bsz, max_len, hk, d = tensors[0].shape
    if q.dim() != 4 or q.shape[0] != bsz or q.shape[3] != d or q.dtype is not torch.bfloat16:
        raise ValueError(f"q must be bf16 [B={bsz}, n, H, D={d}], got {q.dtype} {tuple(q.shape)}")
    n, heads = q.shape[1:3]
    if heads < hk or heads % hk:
        raise ValueError(f"{heads} query heads do not share {hk} key heads")
    lens, len_ptr, len_all = _start(kv_len, bsz, "kv_len")
    window = 0 if window is None else _count(window, "window", 1)
    sink = _count(sink, "sink", 0)
    scale, cap = check_scores(d, heads, scale, cap, slopes)
    index = num = None
    topk = 0
    if chosen is not None:
        index, num = chosen
        if window or sink:
            raise ValueError("chosen blocks take no window and no sink")
        if (index.dim() != 4 or tuple(index.shape[:3]) != (bsz, n, hk) or tuple(num.shape) != (bsz, n, hk)
                or index.dtype is not torch.int32 or num.dtype is not torch.int32 or not 1 <= index.shape[3] <= _lib.SELECT_MAX_BLOCKS):
            raise ValueError(f"chosen must be int32 index [{bsz}, {n}, {hk}, 1 .. {_lib.SELECT_MAX_BLOCKS}] and num [{bsz}, {n}, {hk}], got "
                             f"{index.dtype} {tuple(index.shape)} and {num.dtype} {tuple(num.shape)}")
        index, num, topk = index.contiguous(), num.contiguous(), index.shape[3]
    elif sink and not window:
        raise ValueError("sink needs a window (without one every token is seen)")
    _no_gradient(q, slopes)
    dev = _lib.require_gpu(*tensors, q, slopes, lens, index, num)
    slopes = None if slopes is None else slopes.contiguous()
    if q.numel() == 0:
        return torch.empty_like(q), torch.empty((bsz, heads, n), dtype=torch.float32, device=dev)
    q = _lib.kernel_ready(q)
    if chosen is None and n * (heads // hk) > _FEW_ROWS:
        tokens = max_len if lens is not None else min(max(len_all, 0), max_len)
        k, v = _read(c, dev, None, 0, tokens, torch.bfloat16, (len_ptr, len_all if lens is None else 0), n, window, sink)
        ranges = _make_ranges(bsz, n, tokens, window=window or None, sink=sink, kv_len=len_all if lens is None else lens, device=dev,
                              in_order=True)   # for one call: not worth sorting
        if not 0 <= q.stride(1) <= 1 << 23:
            q = q.clone(memory_format=torch.contiguous_format)
        return _forward(q, k, v, slopes, ranges, scale, cap)
    out = torch.empty((bsz, n, heads, d), dtype=torch.bfloat16, device=dev)
    lse = torch.empty((bsz, heads, n), dtype=torch.float32, device=dev)
    args = _lib.Kv8AttendArgs(c, *_lib.blhd(q), *_lib.blhd(out), lse.data_ptr(), n, heads, len_ptr, len_all, _lib.ptr(index), _lib.ptr(num),
                              topk, window, sink, _lib.ptr(slopes), scale, cap, None)
    size = _lib.lib().wa_kv8_attend_workspace_bytes(args)
    if size:
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        args.workspace = ws.data_ptr()
    _lib.launch("wa_kv8_attend", args, dev)
    return out, lse
