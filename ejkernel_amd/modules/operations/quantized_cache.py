"""The 8-bit paged cache with a scale per block of tokens and head: writing to it and reading from it.

The reference's 8-bit caches have one scale per tensor (``ragged_page_attention_v3``); this cache
has no counterpart there.  Its two arrays:

``kv_cache``   ``[num_pages, 2 * num_kv_heads, page_size, head_dim]`` codes, ``torch.int8``,
               ``torch.float8_e4m3fn`` or ``torch.float8_e5m2``; K of kv head ``j`` at ``2j``, V at
               ``2j + 1``.  The tokens of a page lie together for each head.
``kv_scales``  ``[num_pages, 2 * num_kv_heads, page_size // block]`` float32; an element is its code
               times the scale of its block of ``block`` tokens.

``head_dim`` is a multiple of 16 up to 256, ``page_size`` and ``block`` are powers of two from 4 on.
The attention over it is ``quantized_ragged_page_attention``.
"""

from __future__ import annotations

import ctypes

import torch

from ... import _native

__all__ = ["QuantizedCacheGather", "QuantizedCacheUpdate", "quantized_cache_gather", "quantized_cache_update"]

_CACHE_DTYPES = {torch.int8: _native.RPA_DTYPE_INT8, torch.float8_e4m3fn: _native.RPA_DTYPE_FP8_E4M3,
                 torch.float8_e5m2: _native.RPA_DTYPE_FP8_E5M2}
_VALUE_DTYPES = {torch.bfloat16: _native.RPA_DTYPE_BF16, torch.float32: _native.RPA_DTYPE_F32}


def _check_cache(kv_cache, kv_scales) -> int:
    """Checks the two arrays against each other; returns the tokens a scale covers."""
    if kv_cache.dim() != 4:
        raise ValueError(f"kv_cache must be [num_pages, 2 * num_kv_heads, page_size, head_dim], got {tuple(kv_cache.shape)}")
    if kv_cache.dtype not in _CACHE_DTYPES:
        raise ValueError(f"kv_cache.dtype={kv_cache.dtype} must be int8, float8_e4m3fn or float8_e5m2")
    num_pages, heads, page_size, _ = kv_cache.shape
    if heads % 2 != 0 or heads == 0:
        raise ValueError(f"kv_cache.shape[1]={heads} must be 2 * num_kv_heads")
    if kv_scales.dim() != 3 or kv_scales.dtype != torch.float32 or kv_scales.shape[0] != num_pages or kv_scales.shape[1] != heads:
        raise ValueError(f"kv_scales must be float32 [{num_pages}, {heads}, page_size // block], got {kv_scales.dtype} {tuple(kv_scales.shape)}")
    blocks = kv_scales.shape[2]
    if blocks == 0 or page_size % blocks != 0:
        raise ValueError(f"kv_scales.shape[2]={blocks} must divide page_size={page_size}")
    if not kv_cache.is_contiguous() or not kv_scales.is_contiguous():
        raise ValueError("kv_cache and kv_scales must be contiguous")
    return page_size // blocks


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``[tokens, heads, head_dim]`` as the kernels read it in place: rows of 16-byte pieces; anything else is copied."""
    unit = 16 // t.element_size()
    if t.stride(2) == 1 and t.data_ptr() % 16 == 0 and all(t.shape[k] <= 1 or t.stride(k) % unit == 0 for k in (0, 1)):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strides(t: torch.Tensor) -> tuple[int, int]:
    return (t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0)


def _on_device(op: str, first: torch.Tensor, **others: torch.Tensor) -> torch.device:
    if not first.is_cuda:
        raise RuntimeError(f"{op} needs tensors on a ROCm device (gfx950); there is no CPU implementation in this package.")
    dev = first.device
    for name, t in others.items():
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev}")
    return dev


def _call(entry: str, params, dev: torch.device) -> None:
    """Calls a C entry point on the current stream of ``dev``."""
    fn = getattr(_native.load(), entry)
    if torch.cuda.current_device() == dev.index:
        rc = fn(ctypes.byref(params), torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(ctypes.byref(params), torch.cuda.current_stream(dev).cuda_stream)
    if rc != 0:
        kind = ValueError if rc in (-1, -2) else RuntimeError
        raise kind(f"{entry} refused the call ({rc}): {_native.last_error()}")


class QuantizedCacheUpdate:
    """Kernel object of ``quantized_cache_update``."""

    op_id = "quantized_cache_update"

    def run(self, keys, values, kv_cache, kv_scales, slot_mapping):
        block = _check_cache(kv_cache, kv_scales)
        num_pages, heads, page_size, head_dim = kv_cache.shape
        if keys.dim() != 3 or keys.shape != values.shape or keys.shape[1] != heads // 2 or keys.shape[2] != head_dim:
            raise ValueError(f"keys and values must be [total_tokens, {heads // 2}, {head_dim}], got {tuple(keys.shape)} and {tuple(values.shape)}")
        if keys.dtype not in _VALUE_DTYPES or values.dtype != keys.dtype:
            raise ValueError(f"keys and values must share one dtype, bfloat16 or float32, got {keys.dtype} and {values.dtype}")
        if tuple(slot_mapping.shape) != (keys.shape[0],) or slot_mapping.dtype != torch.int32:
            raise ValueError(f"slot_mapping must be int32 [{keys.shape[0]}], got {slot_mapping.dtype} {tuple(slot_mapping.shape)}")
        if any(t.requires_grad for t in (keys, values, kv_scales)):
            raise NotImplementedError("quantized_cache_update is forward-only; detach the inputs")
        dev = _on_device("quantized_cache_update", kv_cache, keys=keys, values=values, kv_scales=kv_scales, slot_mapping=slot_mapping)
        if keys.shape[0] == 0:
            return kv_cache, kv_scales
        keys, values, slot_mapping = _rows(keys), _rows(values), slot_mapping.contiguous()
        p = _native.RpaQuantUpdateParams()
        p.keys, p.values = keys.data_ptr(), values.data_ptr()
        p.kv_cache, p.kv_scales, p.slot_mapping = kv_cache.data_ptr(), kv_scales.data_ptr(), slot_mapping.data_ptr()
        p.key_token_stride, p.key_head_stride = _strides(keys)
        p.value_token_stride, p.value_head_stride = _strides(values)
        p.total_tokens, p.num_kv_heads, p.head_dim = keys.shape[0], heads // 2, head_dim
        p.page_size, p.scale_block, p.num_pages = page_size, block, num_pages
        p.dtype, p.cache_dtype = _VALUE_DTYPES[keys.dtype], _CACHE_DTYPES[kv_cache.dtype]
        _call("rpa_quant_update_launch", p, dev)
        return kv_cache, kv_scales


class QuantizedCacheGather:
    """Kernel object of ``quantized_cache_gather``."""

    op_id = "quantized_cache_gather"

    def run(self, kv_cache, kv_scales, slot_mapping, *, dtype: torch.dtype = torch.bfloat16):
        block = _check_cache(kv_cache, kv_scales)
        num_pages, heads, page_size, head_dim = kv_cache.shape
        if dtype not in _VALUE_DTYPES:
            raise ValueError(f"dtype={dtype} must be bfloat16 or float32")
        if slot_mapping.dim() != 1 or slot_mapping.dtype != torch.int32:
            raise ValueError(f"slot_mapping must be int32 [total_tokens], got {slot_mapping.dtype} {tuple(slot_mapping.shape)}")
        if kv_scales.requires_grad:
            raise NotImplementedError("quantized_cache_gather is forward-only; detach the inputs")
        dev = _on_device("quantized_cache_gather", kv_cache, kv_scales=kv_scales, slot_mapping=slot_mapping)
        tokens = slot_mapping.shape[0]
        keys = torch.empty((tokens, heads // 2, head_dim), dtype=dtype, device=dev)
        values = torch.empty_like(keys)
        if tokens == 0:
            return keys, values
        slot_mapping = slot_mapping.contiguous()
        p = _native.RpaQuantGatherParams()
        p.kv_cache, p.kv_scales, p.slot_mapping = kv_cache.data_ptr(), kv_scales.data_ptr(), slot_mapping.data_ptr()
        p.keys, p.values = keys.data_ptr(), values.data_ptr()
        p.total_tokens, p.num_kv_heads, p.head_dim = tokens, heads // 2, head_dim
        p.page_size, p.scale_block, p.num_pages = page_size, block, num_pages
        p.dtype, p.cache_dtype = _VALUE_DTYPES[dtype], _CACHE_DTYPES[kv_cache.dtype]
        _call("rpa_quant_gather_launch", p, dev)
        return keys, values


_update = QuantizedCacheUpdate()
_gather = QuantizedCacheGather()


def quantized_cache_update(keys, values, kv_cache, kv_scales, slot_mapping, /):
    """Write the keys and values of new tokens into the 8-bit cache.

    Args:
        keys, values: ``[total_tokens, num_kv_heads, head_dim]`` bfloat16 or float32; views with strides of
            whole 16-byte pieces (of one fused projection, say) are read in place.
        kv_cache, kv_scales: the cache (see the module's text), updated in place.
        slot_mapping: ``[total_tokens]`` int32, ``page * page_size + offset`` of each token; a slot outside the
            pool (-1) skips the token.

    Consecutive tokens in consecutive slots of one block are a run and are written with one scale per head:
    ``s = a / 127`` for int8, the least power of two with ``a <= s * max`` for the float8 types, where ``a`` is
    the run's largest finite magnitude.  A run that begins inside a block keeps the rows before it: ``s`` is
    then at least the block's old scale, and where it is larger the codes of those rows are re-expressed in
    it.  Codes are ``round(x / s)`` with ties to even, decided on the exact quotient; infinities become the
    largest code and NaN becomes 0, so the cache never holds a value that is not finite.  Rows of a block
    behind the run are stale.  A block may be written by one run of a call only: with two, the scale it ends
    with is either's.

    Returns:
        ``(kv_cache, kv_scales)``, the arrays that were passed.
    """
    return _update.run(keys, values, kv_cache, kv_scales, slot_mapping)


def quantized_cache_gather(kv_cache, kv_scales, slot_mapping, /, *, dtype: torch.dtype = torch.bfloat16):
    """Rows of the 8-bit cache as values (a request's context to hand over or to look at).

    Args:
        kv_cache, kv_scales: the cache (see the module's text).
        slot_mapping: ``[total_tokens]`` int32 slots, in any order and number; a slot outside the pool gives zeros.
        dtype: bfloat16 or float32.

    Returns:
        ``(keys, values)``, each ``[total_tokens, num_kv_heads, head_dim]``: code times scale in float32, rounded to ``dtype``.
    """
    return _gather.run(kv_cache, kv_scales, slot_mapping, dtype=dtype)
