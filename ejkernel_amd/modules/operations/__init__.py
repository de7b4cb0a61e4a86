from .block_tables import BlockTables, BuildBlockTables, build_block_tables
from .configs import (
    BaseOperationConfig,
    FwdParams,
    PageAttentionConfig,
    QuantizedRaggedPageAttentionConfig,
    RaggedDecodeAttentionConfig,
    RaggedPageAttentionConfig,
    RaggedPageAttentionv3Config,
)
from .page_attention import PageAttention, page_attention
from .quantized_cache import QuantizedCacheGather, QuantizedCacheUpdate, quantized_cache_gather, quantized_cache_update
from .quantized_ragged_page_attention import QuantizedRaggedPageAttention, quantized_ragged_page_attention
from .ragged_decode_attention import RaggedDecodeAttention, ragged_decode_attention
from .ragged_page_attention import RaggedPageAttention, ragged_page_attention
from .ragged_page_attention_v3 import RaggedPageAttentionv3, ragged_page_attention_v3

__all__ = ['BaseOperationConfig', 'BlockTables', 'BuildBlockTables', 'FwdParams', 'PageAttention', 'PageAttentionConfig', 'QuantizedCacheGather', 'QuantizedCacheUpdate', 'QuantizedRaggedPageAttention', 'QuantizedRaggedPageAttentionConfig', 'RaggedDecodeAttention', 'RaggedDecodeAttentionConfig', 'RaggedPageAttention', 'RaggedPageAttentionConfig', 'RaggedPageAttentionv3', 'RaggedPageAttentionv3Config', 'build_block_tables', 'page_attention', 'quantized_cache_gather', 'quantized_cache_update', 'quantized_ragged_page_attention', 'ragged_decode_attention', 'ragged_page_attention', 'ragged_page_attention_v3']
