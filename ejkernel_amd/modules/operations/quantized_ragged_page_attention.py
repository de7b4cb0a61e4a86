"""Ragged paged attention over an 8-bit cache with a scale per block of tokens and head.

Takes the batch of ``ragged_page_attention`` -- flat queries, context lengths, block tables, query
starts -- and the cache of ``quantized_cache_update``.  Nothing like it is in the reference, whose
8-bit caches have one scale per tensor and round probabilities to the cache's type: here codes are
widened, scales enter the logits and the probabilities in float32, and only the products of
probability and value scale are rounded: to 16 bits in decode steps, to bfloat16 in longer chunks, with
float32 queries not at all.
"""

from __future__ import annotations

import ctypes

import torch

from ... import _native
from .configs import QuantizedRaggedPageAttentionConfig
from .quantized_cache import _VALUE_DTYPES, _call, _check_cache, _check_index_arrays, _current_device, _on_device, _raw_stream, _rows
from .ragged_page_attention import _call_workspace, _sinks_per_q_head

__all__ = ["QuantizedRaggedPageAttention", "quantized_ragged_page_attention"]


_sizes: dict[tuple[int, int, int], int] = {}  # workspace bytes by device, dtype and head_dim, all that they depend on


class QuantizedRaggedPageAttention:
    """Kernel object of ``quantized_ragged_page_attention``."""

    op_id = "quantized_ragged_page_attention"
    _entry = _native.Entry("rpa_quant_fwd_launch", _native.RpaQuantParams)

    def run(self, queries, kv_cache, kv_scales, context_lens, block_tables, query_start_loc, num_seqs, softmax_aux=None, *,
            softmax_scale: float | None = None, logits_soft_cap: float | None = None, sliding_window: int | None = None,
            cfg: QuantizedRaggedPageAttentionConfig):
        cfg.validate()
        num_pages, heads, page_size, head_dim, block, code = _check_cache(kv_cache, kv_scales)
        num_kv_heads = heads // 2
        shape = queries.shape
        if len(shape) != 3 or shape[2] != head_dim:
            raise ValueError(f"queries must be [total_tokens, num_q_heads, {head_dim}], got {tuple(shape)}")
        dtype = _VALUE_DTYPES.get(queries.dtype)
        if dtype is None:
            raise ValueError(f"queries.dtype={queries.dtype} must be bfloat16 or float32")
        total_tokens, num_q_heads, _ = shape
        if num_q_heads == 0 or num_q_heads % num_kv_heads != 0:
            raise ValueError(f"{num_q_heads=} must be divisible by {num_kv_heads=}")
        if block_tables.dim() != 2 or 0 in block_tables.shape:
            raise ValueError(f"block_tables must be [max_num_seqs, pages_per_seq], got {tuple(block_tables.shape)}")
        max_num_seqs, pages_per_seq = block_tables.shape
        if not isinstance(num_seqs, torch.Tensor):
            num_seqs = torch.tensor([int(num_seqs)], dtype=torch.int32, device=queries.device)
        _check_index_arrays(("context_lens", context_lens, max_num_seqs), ("query_start_loc", query_start_loc, max_num_seqs + 1), ("num_seqs", num_seqs, 1))
        if block_tables.dtype != torch.int32:
            raise ValueError(f"block_tables.dtype={block_tables.dtype} must be int32")
        if sliding_window is not None and sliding_window <= 0:
            raise ValueError(f"{sliding_window=} must be positive.")
        if logits_soft_cap is not None and logits_soft_cap == 0.0:
            raise ValueError(f"{logits_soft_cap=} must not be 0.0.")
        if queries.requires_grad or kv_scales.requires_grad:
            raise NotImplementedError("quantized_ragged_page_attention is forward-only; detach the inputs")
        index = _on_device("quantized_ragged_page_attention", ("queries", queries), ("kv_cache", kv_cache), ("kv_scales", kv_scales),
                           ("context_lens", context_lens), ("block_tables", block_tables), ("query_start_loc", query_start_loc), ("num_seqs", num_seqs))
        if _current_device() != index:
            with torch.cuda.device(index):
                return self.run(queries, kv_cache, kv_scales, context_lens, block_tables, query_start_loc, num_seqs, softmax_aux,
                                softmax_scale=softmax_scale, logits_soft_cap=logits_soft_cap, sliding_window=sliding_window, cfg=cfg)
        out = queries.new_empty(shape)
        if total_tokens == 0:
            return out
        queries, address, token_stride, head_stride = _rows(queries, shape)
        context_lens, block_tables, query_start_loc = context_lens.contiguous(), block_tables.contiguous(), query_start_loc.contiguous()
        sinks = None
        if softmax_aux is not None and softmax_aux.shape[-1] > 0:
            sinks = _sinks_per_q_head(softmax_aux.to(queries.device), num_q_heads, num_kv_heads)
        size = _sizes.get((index, dtype, head_dim))
        if size is None:
            size = self._workspace_bytes(index, dtype, head_dim)
        workspace = _call_workspace(queries.device, size, _raw_stream(index))
        _call(self._entry, index, address, kv_cache.data_ptr(), kv_scales.data_ptr(), context_lens.data_ptr(), block_tables.data_ptr(),
              query_start_loc.data_ptr(), num_seqs.data_ptr(), 0 if sinks is None else sinks.data_ptr(), out.data_ptr(),
              workspace.data_ptr(), workspace.numel(), token_stride, head_stride, total_tokens, num_q_heads, num_kv_heads, head_dim, page_size, block,
              num_pages, max_num_seqs, pages_per_seq, 0 if sinks is None else sinks.shape[1],
              head_dim**-0.5 if softmax_scale is None else softmax_scale, 0.0 if logits_soft_cap is None else logits_soft_cap,
              0 if sliding_window is None else min(sliding_window, 2**31 - 1), dtype, code, 0)
        return out

    @staticmethod
    def _workspace_bytes(index: int, dtype: int, head_dim: int) -> int:
        """Asks the library once per device, dtype and head_dim; other dims do not enter the size."""
        p = _native.RpaQuantParams()
        p.num_q_heads = p.num_kv_heads = p.num_pages = p.max_num_seqs = p.pages_per_seq = 1
        p.page_size = p.scale_block = 16
        p.head_dim, p.dtype, p.cache_dtype = head_dim, dtype, _native.RPA_DTYPE_INT8
        size = int(_native.load().rpa_quant_workspace_bytes(ctypes.byref(p)))
        if size == 0:
            raise ValueError(_native.last_error())
        _sizes[(index, dtype, head_dim)] = size
        return size

    def heuristic_cfg(self, inv=None) -> QuantizedRaggedPageAttentionConfig:
        """The work is cut on the device; there is nothing to choose."""
        return QuantizedRaggedPageAttentionConfig()

    def candidate_cfgs(self, inv=None) -> list[QuantizedRaggedPageAttentionConfig]:
        """One implementation, one candidate."""
        return [self.heuristic_cfg(inv)]

    def __call__(self, *args, **kwargs):
        kwargs.setdefault("cfg", self.heuristic_cfg())
        return self.run(*args, **kwargs)


_kernel = QuantizedRaggedPageAttention()
_default_cfg = QuantizedRaggedPageAttentionConfig()


def quantized_ragged_page_attention(
    queries,
    kv_cache,
    kv_scales,
    context_lens,
    block_tables,
    query_start_loc,
    num_seqs,
    softmax_aux=None,
    /,
    *,
    softmax_scale: float | None = None,
    logits_soft_cap: float | None = None,
    sliding_window: int | None = None,
    cfg: QuantizedRaggedPageAttentionConfig | None = None,
):
    """Attention of a mixed prefill + decode batch over the 8-bit paged cache.

    Args:
        queries: ``[total_tokens, num_q_heads, head_dim]`` bfloat16 or float32, all sequences one after another;
            views with strides of whole 16-byte pieces are read in place.
        kv_cache: ``[num_pages, 2 * num_kv_heads, page_size, head_dim]`` int8, float8_e4m3fn or float8_e5m2;
            K of kv head ``j`` at ``2j``, V at ``2j + 1``.  Every value a sequence can see must be finite.
        kv_scales: ``[num_pages, 2 * num_kv_heads, page_size // block]`` float32, finite and not negative where a
            sequence can see the block.
        context_lens: ``[max_num_seqs]`` int32, keys of each sequence including its query tokens.
        block_tables: ``[max_num_seqs, pages_per_seq]`` int32; entries behind a sequence's pages are not read.
        query_start_loc: ``[max_num_seqs + 1]`` int32 cumulative query lengths.
        num_seqs: ``[1]`` int32 tensor (or int), sequences present.
        softmax_aux: optional sink logits ``[num_kv_heads | num_q_heads, n_sinks]`` or ``[n_sinks]``.
        softmax_scale: defaults to ``head_dim ** -0.5``.
        logits_soft_cap: ``cap * tanh(logits / cap)`` before masking.
        sliding_window: keep keys with ``k_pos > q_pos - window``.

    Returns:
        ``[total_tokens, num_q_heads, head_dim]`` in the dtype of ``queries``; rows without a visible key and rows
        at or beyond ``query_start_loc[num_seqs]`` are zero.
    """
    return _kernel.run(queries, kv_cache, kv_scales, context_lens, block_tables, query_start_loc, num_seqs, softmax_aux,
                       softmax_scale=softmax_scale, logits_soft_cap=logits_soft_cap, sliding_window=sliding_window,
                       cfg=_default_cfg if cfg is None else cfg)
