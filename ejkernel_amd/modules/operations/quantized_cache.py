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

import torch

from ... import _native

__all__ = ["QuantizedCacheGather", "QuantizedCacheUpdate", "quantized_cache_gather", "quantized_cache_update"]

_CACHE_DTYPES = {torch.int8: _native.RPA_DTYPE_INT8, torch.float8_e4m3fn: _native.RPA_DTYPE_FP8_E4M3,
                 torch.float8_e5m2: _native.RPA_DTYPE_FP8_E5M2}
_VALUE_DTYPES = {torch.bfloat16: _native.RPA_DTYPE_BF16, torch.float32: _native.RPA_DTYPE_F32}


_raw_stream = torch._C._cuda_getCurrentRawStream  # the handle alone: torch.cuda.current_stream builds an object around it
_current_device = torch._C._cuda_getDevice


def _check_cache(kv_cache, kv_scales) -> tuple[int, int, int, int, int, int]:
    """Checks the two arrays against each other; returns the shape of the cache, the tokens a scale covers and the type's code."""
    shape = kv_cache.shape
    if len(shape) != 4:
        raise ValueError(f"kv_cache must be [num_pages, 2 * num_kv_heads, page_size, head_dim], got {tuple(shape)}")
    code = _CACHE_DTYPES.get(kv_cache.dtype)
    if code is None:
        raise ValueError(f"kv_cache.dtype={kv_cache.dtype} must be int8, float8_e4m3fn or float8_e5m2")
    num_pages, heads, page_size, head_dim = shape
    if heads % 2 != 0 or heads == 0:
        raise ValueError(f"kv_cache.shape[1]={heads} must be 2 * num_kv_heads")
    shape = kv_scales.shape
    if len(shape) != 3 or kv_scales.dtype != torch.float32 or shape[0] != num_pages or shape[1] != heads:
        raise ValueError(f"kv_scales must be float32 [{num_pages}, {heads}, page_size // block], got {kv_scales.dtype} {tuple(shape)}")
    blocks = shape[2]
    if blocks == 0 or page_size % blocks != 0:
        raise ValueError(f"kv_scales.shape[2]={blocks} must divide page_size={page_size}")
    if not kv_cache.is_contiguous() or not kv_scales.is_contiguous():
        raise ValueError("kv_cache and kv_scales must be contiguous")
    return num_pages, heads, page_size, head_dim, page_size // blocks, code


def _rows(t: torch.Tensor, shape) -> tuple[torch.Tensor, int, int, int]:
    """``[tokens, heads, head_dim]`` as the kernels read it in place, rows of 16-byte pieces, with its address and its strides
    between tokens and heads; anything else is copied."""
    address = t.data_ptr()
    if address % 16 == 0 and t.is_contiguous():  # (head_dim is checked behind the C entry)
        return t, address, shape[1] * shape[2], shape[2]
    unit = 16 // t.element_size()
    for _ in range(3):
        token, head, element = t.stride()
        if shape[0] <= 1:
            token = 0
        if shape[1] <= 1:
            head = 0
        if element == 1 and token % unit == 0 and head % unit == 0 and t.data_ptr() % 16 == 0:
            break
        t = t.clone() if t.is_contiguous() else t.contiguous()
    return t, t.data_ptr(), token, head


def _check_index_arrays(*arrays: tuple[str, torch.Tensor, int]) -> None:
    """Name, tensor and length of arrays that are int32 vectors."""
    for name, t, length in arrays:
        if t.shape != (length,):
            raise ValueError(f"{name}.shape={tuple(t.shape)} must be ({length},)")
        if t.dtype != torch.int32:
            raise ValueError(f"{name}.dtype={t.dtype} must be int32")


def _on_device(op: str, *tensors: tuple[str, torch.Tensor]) -> int:
    """Index of the device that all of the tensors are on."""
    first = tensors[0][1]
    index = first.get_device()
    if index < 0:
        raise RuntimeError(f"{op} needs tensors on a ROCm device (gfx950); there is no CPU implementation in this package.")
    for name, t in tensors:
        if t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, expected {first.device}")
    return index


def _call(entry: _native.Entry, index: int, *values) -> None:
    """Calls a C entry point on the current stream of device ``index``."""
    if _current_device() == index:
        entry(_raw_stream(index), *values)
    else:
        with torch.cuda.device(index):
            entry(_raw_stream(index), *values)


class QuantizedCacheUpdate:
    """Kernel object of ``quantized_cache_update``."""

    op_id = "quantized_cache_update"
    _entry = _native.Entry("rpa_quant_update_launch", _native.RpaQuantUpdateParams)

    def run(self, keys, values, kv_cache, kv_scales, slot_mapping):
        num_pages, heads, page_size, head_dim, block, code = _check_cache(kv_cache, kv_scales)
        shape = keys.shape
        if len(shape) != 3 or shape != values.shape or shape[1] != heads // 2 or shape[2] != head_dim:
            raise ValueError(f"keys and values must be [total_tokens, {heads // 2}, {head_dim}], got {tuple(shape)} and {tuple(values.shape)}")
        dtype = _VALUE_DTYPES.get(keys.dtype)
        if dtype is None or values.dtype != keys.dtype:
            raise ValueError(f"keys and values must share one dtype, bfloat16 or float32, got {keys.dtype} and {values.dtype}")
        tokens = shape[0]
        if slot_mapping.shape != (tokens,) or slot_mapping.dtype != torch.int32:
            raise ValueError(f"slot_mapping must be int32 [{tokens}], got {slot_mapping.dtype} {tuple(slot_mapping.shape)}")
        if keys.requires_grad or values.requires_grad or kv_scales.requires_grad:
            raise NotImplementedError("quantized_cache_update is forward-only; detach the inputs")
        index = _on_device("quantized_cache_update", ("kv_cache", kv_cache), ("keys", keys), ("values", values), ("kv_scales", kv_scales), ("slot_mapping", slot_mapping))
        if tokens == 0:
            return kv_cache, kv_scales
        keys, key_address, key_token, key_head = _rows(keys, shape)
        values, value_address, value_token, value_head = _rows(values, shape)
        slot_mapping = slot_mapping.contiguous()
        _call(self._entry, index, key_address, value_address, kv_cache.data_ptr(), kv_scales.data_ptr(), slot_mapping.data_ptr(),
              key_token, key_head, value_token, value_head, tokens, heads // 2, head_dim, page_size, block, num_pages, dtype, code)
        return kv_cache, kv_scales


class QuantizedCacheGather:
    """Kernel object of ``quantized_cache_gather``."""

    op_id = "quantized_cache_gather"
    _entry = _native.Entry("rpa_quant_gather_launch", _native.RpaQuantGatherParams)

    def run(self, kv_cache, kv_scales, slot_mapping, *, dtype: torch.dtype = torch.bfloat16):
        num_pages, heads, page_size, head_dim, block, code = _check_cache(kv_cache, kv_scales)
        kind = _VALUE_DTYPES.get(dtype)
        if kind is None:
            raise ValueError(f"dtype={dtype} must be bfloat16 or float32")
        if slot_mapping.dim() != 1 or slot_mapping.dtype != torch.int32:
            raise ValueError(f"slot_mapping must be int32 [total_tokens], got {slot_mapping.dtype} {tuple(slot_mapping.shape)}")
        if kv_scales.requires_grad:
            raise NotImplementedError("quantized_cache_gather is forward-only; detach the inputs")
        index = _on_device("quantized_cache_gather", ("kv_cache", kv_cache), ("kv_scales", kv_scales), ("slot_mapping", slot_mapping))
        tokens = slot_mapping.shape[0]
        shape = (tokens, heads // 2, head_dim)
        keys = kv_scales.new_empty(shape, dtype=dtype)
        values = torch.empty_like(keys)
        if tokens == 0:
            return keys, values
        slot_mapping = slot_mapping.contiguous()
        _call(self._entry, index, kv_cache.data_ptr(), kv_scales.data_ptr(), slot_mapping.data_ptr(), keys.data_ptr(), values.data_ptr(),
              tokens, heads // 2, head_dim, page_size, block, num_pages, kind, code)
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
