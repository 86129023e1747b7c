"""Hybrid Sparse Attention on MI355X — public API of ``wan/modules/hsa/__init__.py:3-26``."""

from .attention import (
    HSAAttention,
    compress_kv,
    hsa_attention,
    hsa_parameter_names,
    require_trained_hsa,
    resolve_backend,
)
from .kvcache import kv_append, new_block_sums
from .block_sparse import block_sparse_attention, block_sparse_attention_reference, map_to_index
from .decay import decay_linear_attention, decay_linear_step
from .rope import axis_frequencies, rope_axes
from .selected import BlockSelection, attend_selected, select_key_blocks, selected_attention
from .routing import (
    BlockRouting,
    block_attention_map,
    block_mean_pool,
    build_block_routing,
    build_topk_routing,
)

__all__ = [
    "HSAAttention",
    "hsa_attention",
    "compress_kv",
    "resolve_backend",
    "hsa_parameter_names",
    "require_trained_hsa",
    "block_sparse_attention_reference",
    "block_sparse_attention",
    "map_to_index",
    "BlockRouting",
    "build_block_routing",
    "build_topk_routing",
    "block_attention_map",
    "block_mean_pool",
    "kv_append",
    "new_block_sums",
    "rope_axes",
    "axis_frequencies",
    "decay_linear_attention",
    "decay_linear_step",
    "BlockSelection",
    "select_key_blocks",
    "selected_attention",
    "attend_selected",
]
