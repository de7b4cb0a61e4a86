"""Refusals of the operations on the 8-bit cache and of the block tables, before any launch; the restatements' own pins."""

import ctypes
import pathlib
import re

import numpy as np
import pytest
import torch

from ejkernel_amd import _native
from ejkernel_amd.modules import (QuantizedRaggedPageAttention, QuantizedRaggedPageAttentionConfig, build_block_tables, quantized_cache_gather,
                                  quantized_cache_update, quantized_ragged_page_attention)
from oracle import quantized_oracle as oracle

HEADER = pathlib.Path(__file__).resolve().parents[1] / "include" / "rpa_mi355x.h"


@pytest.mark.parametrize("name", ["RpaQuantParams", "RpaQuantUpdateParams", "RpaQuantGatherParams", "RpaBlockTablesParams"])
def test_struct_layouts_match_header_field_order(name):
    text = HEADER.read_text()
    body = re.sub(r"/\*.*?\*/", "", text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")], flags=re.S)
    assert re.findall(r"([a-z_]+)\s*;", body) == [f[0] for f in getattr(_native, name)._fields_]


@pytest.mark.parametrize("kind,dtype", [("e4m3", torch.float8_e4m3fn), ("e5m2", torch.float8_e5m2), ("int8", torch.int8)])
def test_oracle_codes_are_torch_s(kind, dtype):
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    np.testing.assert_array_equal(oracle.VALUES[kind], codes.view(dtype).double().numpy())
    if kind != "int8":
        x = np.random.default_rng(0).standard_normal(20000) * np.exp2(np.random.default_rng(1).uniform(-18, 8, 20000))
        x = np.clip(x, -oracle.QMAX[kind], oracle.QMAX[kind]).astype(np.float32)
        np.testing.assert_array_equal(oracle.nearest_codes(x.astype(np.float64), kind), torch.from_numpy(x).to(dtype).view(torch.uint8).numpy())


@pytest.mark.parametrize("kind", ["int8", "e4m3", "e5m2"])
def test_oracle_scales_are_the_least_that_hold_the_run(kind):
    for a in (1e-45, 2.0**-126, 0.37, 1.0, 127.0, 448.0, 449.0, 57344.0, 57345.0, 3.4e38):
        s = float(oracle.fresh_scale(a, kind))
        assert s >= 2.0**-126 and (s * oracle.QMAX[kind] >= a * (1 - 2.0**-23))
        if kind != "int8":
            assert np.log2(s) % 1 == 0 and (s == 2.0**-126 or s / 2 * oracle.QMAX[kind] < a)


def test_oracle_attention_is_a_softmax():
    rng = np.random.default_rng(2)
    codes = rng.integers(-127, 128, size=(3, 2, 4, 16)).astype(np.int8).view(np.uint8)
    scales = rng.uniform(0.01, 0.02, size=(3, 2, 1)).astype(np.float32)
    q = rng.standard_normal((2, 2, 16))
    out, _, _ = oracle.attention(q, codes, scales, [7], np.array([[2, 0]]), [0, 2], 1, "int8")
    rows = oracle.cache_values(codes, scales, "int8")[[2, 0]].transpose(1, 0, 2, 3).reshape(2, 8, 16)
    x = torch.from_numpy(q[1, 0] @ rows[0, :7].T / 4)
    np.testing.assert_allclose(out[1, 0], torch.softmax(x, 0).numpy() @ rows[1, :7], rtol=1e-12)


def cache(pages=2, heads=2, page=16, dim=64, block=16, dtype=torch.int8):
    return torch.zeros((pages, 2 * heads, page, dim), dtype=dtype), torch.zeros((pages, 2 * heads, page // block))


def attention_args(**kw):
    c, s = cache(**kw)
    q = torch.zeros((3, 4, c.shape[3]), dtype=torch.bfloat16)
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return [q, c, s, i(5, 6), torch.zeros((2, 2), dtype=torch.int32), i(0, 1, 3), i(2)]


def test_attention_refuses_what_it_does_not_take():
    good = attention_args()
    with pytest.raises(RuntimeError, match="ROCm device"):
        quantized_ragged_page_attention(*good)
    for at, value, match in ((0, good[0][0], "queries must be"), (0, good[0].half(), "dtype"), (0, good[0][..., :32], "queries must be"),
                             (0, good[0][:, :3], "divisible"), (1, good[1][0], "kv_cache must be"), (1, good[1].float(), "int8"),
                             (1, good[1][:, :3], "2 \\* num_kv_heads"), (2, good[2].double(), "float32"), (2, good[2][:1], "kv_scales"),
                             (2, torch.zeros(2, 4, 3), "divide"), (3, good[3].long(), "int32"), (3, good[3][:1], "context_lens"),
                             (4, good[4][0], "block_tables"), (4, good[4].long(), "int32"), (5, good[5][:2], "query_start_loc"),
                             (6, good[5], "num_seqs"), (1, good[1].transpose(2, 3).contiguous().transpose(2, 3), "contiguous")):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError, match=match):
            quantized_ragged_page_attention(*args)
    for kw, match in ((dict(sliding_window=0), "sliding_window"), (dict(logits_soft_cap=0.0), "soft_cap")):
        with pytest.raises(ValueError, match=match):
            quantized_ragged_page_attention(*good, **kw)
    with pytest.raises(NotImplementedError):
        quantized_ragged_page_attention(good[0].requires_grad_(), *good[1:])
    with pytest.raises(ValueError, match="platform"):
        quantized_ragged_page_attention(*attention_args(), cfg=QuantizedRaggedPageAttentionConfig(platform="tpu"))
    assert QuantizedRaggedPageAttention().candidate_cfgs() == [QuantizedRaggedPageAttentionConfig()]


def test_cache_operations_refuse_what_they_do_not_take():
    c, s = cache()
    k, slots = torch.zeros((3, 2, 64)), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device"):
        quantized_cache_update(k, k, c, s, slots)
    with pytest.raises(RuntimeError, match="ROCm device"):
        quantized_cache_gather(c, s, slots)
    for args, match in (((k[:, :1], k[:, :1], c, s, slots), "keys and values must be"), ((k, k[:2], c, s, slots), "keys and values must be"),
                        ((k.half(), k.half(), c, s, slots), "dtype"), ((k, k.bfloat16(), c, s, slots), "dtype"), ((k, k, c, s, slots.long()), "slot_mapping"),
                        ((k, k, c, s, slots[:2]), "slot_mapping"), ((k, k, c, s.transpose(0, 1), slots), "kv_scales")):
        with pytest.raises(ValueError, match=match):
            quantized_cache_update(*args)
    for args, kw, match in (((c, s, slots.long()), {}, "slot_mapping"), ((c, s, slots), dict(dtype=torch.float16), "dtype"), ((c, s, slots[None]), {}, "slot_mapping")):
        with pytest.raises(ValueError, match=match):
            quantized_cache_gather(*args, **kw)
    with pytest.raises(NotImplementedError):
        quantized_cache_update(k.clone().requires_grad_(), k, c, s, slots)


def test_block_tables_refuse_what_they_do_not_take():
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    good, kw = [i(3), i(3), i(3, 4), i(9), i(2), i(1)], dict(page_size=16, total_tokens=5)
    with pytest.raises(RuntimeError, match="ROCm device"):
        build_block_tables(*good, **kw)
    for at, value, match in ((0, i(2), "query_lens"), (0, i(3).long(), "int32"), (1, i(4), "cached_lens"), (2, i(3), "block_tables"), (2, i(3, 0), "block_tables"),
                             (2, i(4, 3).T, "contiguous"), (3, i(0), "free_pages"), (3, i(18)[::2], "contiguous"), (4, i(3), "free_state"), (5, i(2), "num_seqs")):
        args = list(good)
        args[at] = value
        with pytest.raises(ValueError, match=match):
            build_block_tables(*args, **kw)
    for bad in (dict(page_size=0), dict(total_tokens=-1), dict(page_size=2**31), dict(total_tokens=2**31)):
        with pytest.raises(ValueError):
            build_block_tables(*good, **(kw | bad))


def filled(name):
    """Params whose dims are right and whose pointers are aligned; nothing is launched in these tests."""
    p = getattr(_native, name)()
    for field, kind in p._fields_:
        if kind is ctypes.c_void_p:
            setattr(p, field, 0x1000)
    if name == "RpaBlockTablesParams":
        p.max_num_seqs, p.pages_per_seq, p.num_free_slots, p.page_size, p.total_tokens = 3, 4, 9, 16, 5
        return p
    p.total_tokens, p.num_kv_heads, p.head_dim, p.page_size, p.scale_block, p.num_pages, p.cache_dtype = 3, 2, 64, 16, 8, 4, _native.RPA_DTYPE_INT8
    if name == "RpaQuantParams":
        p.num_q_heads, p.max_num_seqs, p.pages_per_seq, p.softmax_scale = 4, 2, 2, 0.1
        p.query_token_stride, p.query_head_stride = 256, 64
        p.workspace_bytes = 0
    if name == "RpaQuantUpdateParams":
        p.key_token_stride, p.key_head_stride, p.value_token_stride, p.value_head_stride = 128, 64, 128, 64
    return p


ENTRY = {"RpaQuantParams": "rpa_quant_fwd_launch", "RpaQuantUpdateParams": "rpa_quant_update_launch", "RpaQuantGatherParams": "rpa_quant_gather_launch"}


@pytest.mark.parametrize("name", ENTRY)
def test_c_entry_points_check_their_arguments(name):
    lib = _native.load()
    launch = getattr(lib, ENTRY[name])
    assert launch(None, None) == -1
    for field, value, rc in (("num_kv_heads", 0, -1), ("num_pages", 0, -1), ("total_tokens", -1, -1), ("head_dim", 72, -2), ("head_dim", 0, -2), ("head_dim", 272, -2),
                             ("page_size", 24, -2), ("page_size", 2, -2), ("page_size", 65536, -2), ("scale_block", 2, -2), ("scale_block", 12, -2),
                             ("scale_block", 32, -2), ("num_pages", 1 << 28, -2), ("dtype", 2, -1), ("cache_dtype", 0, -1), ("cache_dtype", 9, -1),
                             ("kv_cache", None, -1), ("kv_scales", None, -1), ("kv_cache", 0x1008, -1), ("kv_scales", 0x1002, -1)):
        p = filled(name)
        setattr(p, field, value)
        assert launch(ctypes.byref(p), None) == rc, (field, value, lib.rpa_last_error())
        assert lib.rpa_last_error()
    p = filled(name)
    p.total_tokens, p.kv_cache = 0, None
    assert launch(ctypes.byref(p), None) == 0  # nothing to do


def test_c_attention_arguments():
    lib = _native.load()
    size = lib.rpa_quant_workspace_bytes(ctypes.byref(filled("RpaQuantParams")))
    assert size >= 256 and lib.rpa_quant_workspace_bytes(None) == 0
    for field, value, rc in (("num_q_heads", 3, -1), ("max_num_seqs", 0, -1), ("pages_per_seq", 0, -1), ("pages_per_seq", (1 << 26) + 1, -2), ("sliding_window", -1, -1), ("softmax_scale", float("nan"), -1),
                             ("logits_soft_cap", float("inf"), -1), ("flags", 1, -1), ("num_sinks", -1, -1), ("query_token_stride", 100, -1),
                             ("query_head_stride", -64, -1), ("queries", 0x1004, -1), ("out", None, -1), ("workspace", None, -3), ("workspace_bytes", size - 1, -3),
                             ("workspace", 0x1010, -3)):
        p = filled("RpaQuantParams")
        p.workspace_bytes = size
        setattr(p, field, value)
        assert lib.rpa_quant_fwd_launch(ctypes.byref(p), None) == rc, (field, value, lib.rpa_last_error())


def test_c_block_table_arguments():
    lib = _native.load()
    assert lib.rpa_block_tables_launch(None, None) == -1
    for field, value in (("max_num_seqs", 0), ("pages_per_seq", 0), ("num_free_slots", 0), ("page_size", 0), ("total_tokens", -1), ("query_lens", None),
                         ("block_tables", 0x1002), ("scratch", 0x1004), ("slot_mapping", None), ("free_state_out", None)):
        p = filled("RpaBlockTablesParams")
        setattr(p, field, value)
        assert lib.rpa_block_tables_launch(ctypes.byref(p), None) == -1, (field, value)


def test_pages_of_two_gigabytes_are_refused():
    lib = _native.load()
    for name, entry in ENTRY.items():
        p = filled(name)
        p.num_kv_heads, p.page_size, p.head_dim = 128, 32768, 256  # 2**31 bytes
        if name == "RpaQuantParams":
            p.num_q_heads = 128
        assert getattr(lib, entry)(ctypes.byref(p), None) == -2
        assert b"page" in lib.rpa_last_error()


@pytest.mark.parametrize("name", ["RpaQuantParams", "RpaQuantUpdateParams", "RpaQuantGatherParams", "RpaBlockTablesParams"])
def test_packed_values_are_the_struct(name):
    """Entry packs the values in order into the bytes that setting the fields one by one gives."""
    params = getattr(_native, name)
    p, values = params(), []
    for k, (field, kind) in enumerate(params._fields_):
        value = 0.5 + k if kind is ctypes.c_float else 1000 + k
        setattr(p, field, value)
        values.append(value)
    entry = _native.Entry("unused", params)
    assert entry.layout.pack(*values) == bytes(p)
    for k, (field, kind) in enumerate(params._fields_):
        if kind is ctypes.c_int32:
            with pytest.raises(ValueError, match="out of range"):
                _native.Entry("rpa_quant_fwd_launch", params)(0, *values[:k], 2**31, *values[k + 1:])


def test_workspace_has_a_place_for_every_state_of_a_cut():
    """Two states of a tile's rows for each of two workgroups per compute unit, at every width: rows are bf16, fp32."""
    lib = _native.load()
    p = filled("RpaQuantParams")
    for dim, padded, rows in ((16, 64, (256, 128)), (64, 64, (256, 128)), (96, 128, (192, 128)), (128, 128, (192, 128)), (144, 256, (128, 64)), (256, 256, (128, 64))):
        for dtype, own in zip((_native.RPA_DTYPE_BF16, _native.RPA_DTYPE_F32), rows):
            p.head_dim, p.dtype = dim, dtype
            size = lib.rpa_quant_workspace_bytes(ctypes.byref(p))
            per_slot = (16 + own) * (padded * 4 + 8)
            slots, rest = divmod(size - (1 << 20), per_slot)
            assert rest == 0 and slots >= 2 * 16, (dim, dtype, size)


def test_counts_beyond_2_30_are_refused():
    lib = _native.load()
    for name, entry in (*ENTRY.items(), ("RpaBlockTablesParams", "rpa_block_tables_launch")):
        for field in ("total_tokens", "max_num_seqs", "num_free_slots"):
            p = filled(name)
            if hasattr(p, field):
                setattr(p, field, (1 << 30) + 1)
                assert getattr(lib, entry)(ctypes.byref(p), None) == -2, (name, field, lib.rpa_last_error())
