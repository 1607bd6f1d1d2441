"""gki -- MI355X (gfx950) block-sparse StreamingLLM FlashAttention.

Host side of the graph-kernel-injection hot path: StreamingLLM masks, GPU
kept-block lists, the autograd bridge over the HIP kernels in
``libgki_bsa.so``, and the torch.fx pass that injects it.
"""

from .cross import cross_attention
from .fx_pass import (
    BlockSparseAttentionInjector,
    InjectionConfig,
    SingleLayerTransformer,
    StandardAttention,
    _InjectedTritonAttention,
    pretty_print_graph,
)
from .kv_cache import StreamingKVCache
from .lists import BlockLists, build_block_lists, clear_schedule_cache
from .masks import StreamingMaskSpec, make_dense_mask, make_streaming_mask, streaming_token_mask
from .ops import _BlockSparseFlashAttention, block_sparse_attention
from .paged import PagedKVCache, PageTable, TokenBatch
from .reference import reference_block_sparse_attention
from .rotary import MultiAxisRotary

__all__ = [
    "BlockLists",
    "BlockSparseAttentionInjector",
    "InjectionConfig",
    "MultiAxisRotary",
    "PageTable",
    "PagedKVCache",
    "SingleLayerTransformer",
    "StandardAttention",
    "StreamingKVCache",
    "StreamingMaskSpec",
    "TokenBatch",
    "block_sparse_attention",
    "build_block_lists",
    "clear_schedule_cache",
    "cross_attention",
    "make_dense_mask",
    "make_streaming_mask",
    "pretty_print_graph",
    "reference_block_sparse_attention",
    "streaming_token_mask",
]
