"""Public operation API, importable the way ``ejkernel.modules`` is
(ejkernel/modules/__init__.py:68-70,88-89)."""

from .operations import (
    BaseOperationConfig,
    BlockTables,
    BuildBlockTables,
    FwdParams,
    PageAttention,
    PageAttentionConfig,
    QuantizedCacheGather,
    QuantizedCacheUpdate,
    QuantizedRaggedPageAttention,
    QuantizedRaggedPageAttentionConfig,
    RaggedDecodeAttention,
    RaggedDecodeAttentionConfig,
    RaggedPageAttention,
    RaggedPageAttentionConfig,
    RaggedPageAttentionv3,
    RaggedPageAttentionv3Config,
    build_block_tables,
    page_attention,
    quantized_cache_gather,
    quantized_cache_update,
    quantized_ragged_page_attention,
    ragged_decode_attention,
    ragged_page_attention,
    ragged_page_attention_v3,
)

__all__ = ['BaseOperationConfig', 'BlockTables', 'BuildBlockTables', 'FwdParams', 'PageAttention', 'PageAttentionConfig', 'QuantizedCacheGather', 'QuantizedCacheUpdate', 'QuantizedRaggedPageAttention', 'QuantizedRaggedPageAttentionConfig', 'RaggedDecodeAttention', 'RaggedDecodeAttentionConfig', 'RaggedPageAttention', 'RaggedPageAttentionConfig', 'RaggedPageAttentionv3', 'RaggedPageAttentionv3Config', 'build_block_tables', 'page_attention', 'quantized_cache_gather', 'quantized_cache_update', 'quantized_ragged_page_attention', 'ragged_decode_attention', 'ragged_page_attention', 'ragged_page_attention_v3']
