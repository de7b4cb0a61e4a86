"""The operators around the 8-bit paged cache, as they are measured: cases, inputs, plain forms and kernels.

Four operators of one serving step: ``build_block_tables`` (block tables and slot maps from request lengths),
``quantized_cache_update`` (new keys and values into an 8-bit cache with a scale per block of tokens and head),
``quantized_cache_gather`` (rows of that cache as values) and ``quantized_ragged_page_attention`` (attention over it).
A case names its operator in ``"op"``; lengths are drawn from the case alone, data from the seed.
"""

import math

import numpy as np
import torch

own = False

_QMAX = {"int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}
_CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_TYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases


def _attention(name, decodes, step, chunks, chunk, context, q_heads, kv_heads, head_dim, page, block, cache, dtype="bf16",
               window=0, cap=0.0, sinks=0, lens=1):
    return {"name": name, "op": "attention", "decodes": decodes, "step": step, "chunks": chunks, "chunk": chunk, "context": context,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "block": block, "cache": cache,
            "dtype": dtype, "window": window, "cap": cap, "sinks": sinks, "lens": lens}


def _update(name, seqs, new, prior, kv_heads, head_dim, page, block, cache, dtype="bf16", lens=1):
    return {"name": name, "op": "update", "seqs": seqs, "new": new, "prior": prior, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "block": block, "cache": cache, "dtype": dtype, "lens": lens}


def _gather(name, tokens, kv_heads, head_dim, page, block, cache, dtype="bf16", lens=1):
    return {"name": name, "op": "gather", "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "block": block, "cache": cache, "dtype": dtype, "lens": lens}


def _tables(name, seqs, chunks, chunk, context, page, ended, scarce=False, lens=1):
    return {"name": name, "op": "tables", "seqs": seqs, "chunks": chunks, "chunk": chunk, "context": context, "page": page,
            "ended": ended, "scarce": scarce, "lens": lens}


def listed():
    return [
        # the smallest decode step (8 requests of up to 512 keys): latency
        _attention("decode_small", 8, 1, 0, 0, 512, 8, 2, 128, 16, 16, "int8"),
        # a full decode batch of an 8B model with grouped heads: the stream of the cache
        _attention("decode_llama3_8b", 256, 1, 0, 0, 8192, 32, 8, 128, 16, 16, "int8"),
        # chunked prefill of 16 requests, ragged chunks: the matrix products
        _attention("prefill_chunks", 0, 1, 16, 512, 4096, 32, 8, 128, 32, 32, "e4m3"),
        # local attention with a soft cap, four tokens a step (speculative decoding), wide heads
        _attention("gemma2_local", 64, 4, 0, 0, 8192, 16, 8, 256, 16, 16, "e5m2", window=4096, cap=50.0),
        # a mixed batch in fp32 with sinks, heads of 96 and scales for 8 tokens
        _attention("mixed_head_dim_96", 56, 1, 8, 128, 2048, 32, 8, 96, 32, 8, "int8", dtype="fp32", sinks=2),
        # one token of each of 256 requests into half-filled blocks, read back
        _update("update_decode", 256, 1, 8191, 8, 128, 16, 16, "int8"),
        # the tokens of 16 prefill chunks, read back
        _update("update_prefill", 16, 512, 4096, 8, 128, 32, 32, "e4m3"),
        # ragged pieces in fp32 that begin inside small blocks, read back
        _update("update_head_dim_96", 56, 33, 2048, 8, 96, 32, 8, "int8", dtype="fp32"),
        # one request's context handed over
        _gather("gather_context", 32768, 8, 128, 16, 16, "e4m3"),
        # a few rows in fp32 for a look at them
        _gather("gather_few", 300, 2, 64, 16, 4, "int8", dtype="fp32"),
        # bookkeeping of a decode step: one token for each of 256 requests, some of them ended
        _tables("tables_decode", 256, 0, 0, 8192, 16, 5),
        # bookkeeping of a large mixed step with prefill chunks, short of pages at its end
        _tables("tables_mixed", 2048, 64, 1024, 4096, 16, 100, scarce=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "update", "gather", "tables"))
    lens = rng.randrange(1 << 30)
    cache, dtype = rng.choice(("int8", "e4m3", "e5m2")), rng.choice(("bf16", "bf16", "bf16", "fp32"))
    page = rng.choice((4, 8, 16, 32, 64, 128))
    block = rng.choice([b for b in (4, 8, 16, 32, 64, 128) if b <= page])
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    if op == "attention":
        head_dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
        q_heads = kv_heads * rng.choice((1, 3, 4, 7, 8))
        more = dict(dtype=dtype, window=rng.choice((0, 0, 0, _log(rng, 1, 4096))), cap=rng.choice((0.0, 0.0, 0.0, 30.0)),
                    sinks=rng.choice((0, 0, 0, 1, 3)), lens=lens)
        kind = rng.randrange(3)
        decodes = _log(rng, 1, 96) if kind != 1 else 0
        chunks = _log(rng, 1, 8) if kind != 0 else 0
        case = _attention("", decodes, rng.choice((1, 1, 2)), chunks, _log(rng, 2, 300) if chunks else 0,
                          _log(rng, 1, 16384 // (1 if decodes <= 32 and kind == 0 else 8)), q_heads, kv_heads, head_dim, page, block, cache, **more)
    elif op == "update":
        case = _update("", _log(rng, 1, 200), _log(rng, 1, 40), _log(rng, 1, 2000), kv_heads,
                       rng.choice((64, 80, 96, 128, 192, 256)), page, block, cache, dtype, lens)
    elif op == "gather":
        case = _gather("", _log(rng, 1, 20000), kv_heads, rng.choice((64, 80, 96, 128, 192, 256)), page, block, cache, dtype, lens)
    else:
        seqs = _log(rng, 1, 2000)
        chunks = min(seqs, rng.choice((0, _log(rng, 1, 60))))
        case = _tables("", seqs, chunks, _log(rng, 2, 1000) if chunks else 0, _log(rng, 1, 4096), page, seqs // rng.choice((5, 20, 100)),
                       rng.choice((False, False, True)), lens)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ inputs


def _lengths(case):
    """(new tokens, keys with them) of every sequence of an attention case, from the case alone."""
    rng = np.random.Generator(np.random.PCG64(case["lens"]))
    n, c = case["decodes"], case["chunks"]
    q = np.full(n, case["step"], np.int64)
    kv = np.maximum(rng.integers(case["context"] // 16 + 1, case["context"] + 1, size=n), q) if n else q
    if c:
        qc = rng.integers(max(1, case["chunk"] // 2), case["chunk"] + 1, size=c)
        q = np.concatenate([q, qc])
        kv = np.concatenate([kv, rng.integers(0, case["context"] + 1, size=c) + qc])
    order = rng.permutation(n + c)
    return q[order], kv[order]


def _codes(shape, cache, gen):
    """Random codes of the 8-bit type, as a cache of normally distributed values holds them."""
    out = torch.empty(shape, dtype=_CODE[cache], device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        x = torch.randn(min(1 << 28, flat.numel() - at), generator=gen, device="cuda")
        flat[at:at + x.numel()] = (x * 42.0).round_().clamp_(-127, 127).to(torch.int8) if cache == "int8" else x.mul_(_QMAX[cache] / 8).to(_CODE[cache])
    return out


def _scales(shape, cache, gen):
    """Scales of blocks whose values have a standard deviation between a half and two; powers of two for the floating types."""
    r = torch.rand(shape, generator=gen, device="cuda")
    if cache == "int8":
        return (0.5 + 1.5 * r) / 42.0
    return torch.where(r < 0.5, 4.0, 8.0) / (_QMAX[cache] / 1.75)


def _tensor(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _pages(counts, columns, pool, rng):
    """Block tables over a scattered pool: sequence s owns counts[s] pages, the entries behind them name none."""
    table = np.full((len(counts), columns), -1, np.int64)
    at = np.arange(columns)[None, :] < np.asarray(counts)[:, None]
    table[at] = rng.permutation(pool)[: int(at.sum())]
    return table


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.Generator(np.random.PCG64(seed))
    s = {"case": case}
    if case["op"] == "tables":
        return _prepare_tables(case, rng, s)
    heads, page, block, dim = 2 * case["kv_heads"], case["page"], case["block"], case["head_dim"]
    dtype = _TYPE[case["dtype"]]
    if case["op"] == "attention":
        q, kv = _lengths(case)
        counts = -(-kv // page)
        pool, columns = int(counts.sum()) + 3, int(counts.max()) + 1
        s["tables"] = _tensor(_pages(counts, columns, pool, rng))
        s["lens"], s["start"] = _tensor(kv), _tensor(np.concatenate([[0], np.cumsum(q)]))
        s["count"] = _tensor([len(q)])
        s["queries"] = torch.randn((int(q.sum()), case["q_heads"], dim), generator=gen, device="cuda").to(dtype)
        s["sinks"] = torch.randn((case["q_heads"], case["sinks"]), generator=gen, device="cuda") if case["sinks"] else None
        s["longest"], s["keys"] = int(q.max()), int(kv.max())
    elif case["op"] == "update":
        new, prior = _update_lengths(case)
        counts = -(-(prior % page + new) // page)  # the pages that the step touches: the pool is not much larger
        pool = int(counts.sum()) + 1
        table = _pages(counts, int(counts.max()), pool, rng)
        pos = [p % page + np.arange(n) for p, n in zip(prior, new)]
        slots = [table[i, x // page] * page + x % page for i, x in enumerate(pos)]
        s["slots"] = _tensor(np.concatenate(slots + [np.full(3, -1, np.int64)]))  # three padding tokens
        t = s["slots"].numel()
        fused = torch.randn((t, heads, dim), generator=gen, device="cuda")
        fused = (fused * torch.exp(0.5 * torch.randn((t, 1, 1), generator=gen, device="cuda"))).to(dtype)
        s["new_keys"], s["new_values"] = fused[:, : heads // 2], fused[:, heads // 2:]  # views of one projection's output
        s["every"] = torch.arange(pool * page, dtype=torch.int32, device="cuda")
    else:
        pool = -(-case["tokens"] // page) + 2
        s["slots"] = _tensor(rng.permutation(pool)[: pool - 1, None] * page + np.arange(page)[None, :]).reshape(-1)[: case["tokens"]].clone()
    s["cache"] = _codes((pool, heads, page, dim), case["cache"], gen)
    s["scales"] = _scales((pool, heads, page // block), case["cache"], gen)
    return s


def _update_lengths(case):
    rng = np.random.Generator(np.random.PCG64(case["lens"]))
    new = rng.integers(max(1, case["new"] // 2), case["new"] + 1, size=case["seqs"])
    return new, rng.integers(0, case["prior"] + 1, size=case["seqs"])


def _tables_lengths(case):
    rng = np.random.Generator(np.random.PCG64(case["lens"]))
    n = case["seqs"]
    new = np.ones(n, np.int64)
    cached = rng.integers(0, case["context"] + 1, size=n)
    order = rng.permutation(n)
    for k in order[: case["chunks"]]:
        new[k] = rng.integers(1, case["chunk"] + 1)
    new[order[case["chunks"]: case["chunks"] + case["ended"]]] = -1
    return new, cached


def _prepare_tables(case, rng, s):
    new, cached = _tables_lengths(case)
    page, n = case["page"], case["seqs"]
    columns = -(-(case["context"] + max(1, case["chunk"])) // page)
    have = -(-cached // page)
    need = np.where(new > 0, -(-(cached + new) // page) - have, 0)
    spare = int(need.sum()) * 7 // 8 if case["scarce"] else int(need.sum()) + 10
    pool = int(have.sum()) + spare
    ids = rng.permutation(pool)
    table = np.full((n, columns), -1, np.int64)
    table[np.arange(columns)[None, :] < have[:, None]] = ids[: int(have.sum())]
    head = int(rng.integers(0, pool))
    ring = np.full(pool, -1, np.int64)  # the free pages lie in a ring of as many places as the pool has pages
    ring[(head + np.arange(spare)) % pool] = ids[int(have.sum()):]
    s["new"], s["cached"], s["tables"], s["ring"] = _tensor(new), _tensor(cached), _tensor(table), _tensor(ring)
    s["state"], s["count"] = _tensor([head, spare]), _tensor([n])
    s["tokens"] = int(np.maximum(new, 0).sum()) + 5  # five padding rows
    return s


# ------------------------------------------------------------------------------------------------ one pass


def run(s):
    case = s["case"]
    return {"attention": _run_attention, "update": _run_update, "gather": _run_gather, "tables": _run_tables}[case["op"]](s, case)


def _run_attention(s, case):
    window, cap = case["window"] or None, case["cap"] or None
    if own:
        from ejkernel_amd.modules import quantized_ragged_page_attention

        return quantized_ragged_page_attention(s["queries"], s["cache"], s["scales"], s["lens"], s["tables"], s["start"], s["count"],
                                               s["sinks"], logits_soft_cap=cap, sliding_window=window)
    n, longest, keys = s["lens"].numel(), s["longest"], s["keys"]
    page, block, dim, kv_heads = case["page"], case["block"], case["head_dim"], case["kv_heads"]
    group = case["q_heads"] // kv_heads
    pages = -(-keys // page)
    ids = s["tables"][:, :pages].long().clamp(min=0)
    values = s["cache"][ids].float() * s["scales"][ids].repeat_interleave(block, dim=3)[..., None]
    values = values.permute(0, 2, 1, 3, 4).reshape(n, 2 * kv_heads, pages * page, dim)
    k, v = values[:, 0::2], values[:, 1::2]
    start, lens = s["start"].long(), s["lens"].long()
    q_lens = start[1:] - start[:-1]
    at = start[:-1, None] + torch.arange(longest, device="cuda")
    rows = s["queries"].float()[at.clamp(max=s["queries"].shape[0] - 1)]
    q = rows.view(n, longest, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, group * longest, dim)
    x = torch.matmul(q * dim**-0.5, k.transpose(-1, -2).contiguous())
    if cap:
        x = cap * torch.tanh(x / cap)
    pos = (lens - q_lens)[:, None] + torch.arange(longest, device="cuda")
    key = torch.arange(pages * page, device="cuda")
    seen = (key <= pos[..., None]) & (key < lens[:, None, None])
    if window:
        seen &= key > pos[..., None] - window
    seen = seen[:, None, None]
    x = x.view(n, kv_heads, group, longest, -1).masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    sinks = None if s["sinks"] is None else s["sinks"].view(1, kv_heads, group, 1, -1)
    if sinks is not None:
        top = torch.maximum(top, sinks.amax(-1, keepdim=True))
    top = top.clamp(min=-3e38)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top).sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kv_heads, group * longest, -1), v).view(n, kv_heads, group, longest, dim)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, longest, case["q_heads"], dim)
    token = torch.arange(s["queries"].shape[0], device="cuda")
    seq = torch.searchsorted(start[1:], token, right=True)
    return o[seq, token - start[seq]].to(s["queries"].dtype)


def _run_update(s, case):
    """The update, and every row of the pool as values: the state that the update leaves."""
    if own:
        from ejkernel_amd.modules import quantized_cache_gather, quantized_cache_update

        cache, scales = quantized_cache_update(s["new_keys"], s["new_values"], s["cache"], s["scales"], s["slots"])
        return quantized_cache_gather(cache, scales, s["every"], dtype=s["new_keys"].dtype), scales
    cache, scales, block, qmax = s["cache"], s["scales"], case["block"], _QMAX[case["cache"]]
    pool, heads, page, dim = cache.shape
    per = page // block
    slot = s["slots"].long()
    real = slot >= 0
    x = torch.stack([s["new_keys"], s["new_values"]], dim=2).reshape(-1, heads, dim).float()
    into = torch.where(real, slot // block, pool * per)  # block of every token; the padding has one of its own
    size = x.abs().amax(-1)
    amax = torch.zeros((pool * per + 1, heads), device="cuda").index_reduce_(0, into, size, "amax")
    first = torch.full((pool * per + 1,), block, device="cuda").index_reduce_(0, into, slot % block, "amin")
    amax, first = amax[:-1].view(pool, per, heads).transpose(1, 2), first[:-1].view(pool, 1, per)
    if case["cache"] == "int8":
        fresh = torch.where(amax > 0, (amax / qmax).clamp(min=2.0**-126), 0.0)
    else:  # the least power of two that keeps amax within the type's range
        fresh = _binade(amax.double()) / (qmax / 1.75)
        fresh = torch.where(fresh * qmax < amax.double(), 2.0 * fresh, fresh)
        fresh = torch.where(amax > 0, fresh.clamp(min=2.0**-126), 0.0).float()
    touched, inside = first < block, (first > 0) & (first < block)
    scale = torch.where(touched, torch.maximum(fresh, torch.where(inside, scales, 0.0)), scales)
    grown = inside & (scale > scales)
    old = cache.view(pool, heads, per, block, dim)
    again = _round(old.double() * (scales.double() / scale.double().clamp(min=1e-300))[..., None, None], case["cache"])
    before = torch.arange(block, device="cuda").view(1, 1, 1, block, 1) < first[..., None, None]
    bits = torch.where(grown[..., None, None] & before, again.view(torch.int8), old.view(torch.int8))
    at = torch.where(real, slot, 0)
    own_scale = scale[at // page, :, at % page // block]
    code = _round(x.double() / own_scale.double().clamp(min=1e-300)[..., None], case["cache"]).view(torch.int8)
    bits = bits.reshape(pool, heads, page, dim).permute(0, 2, 1, 3).reshape(pool * page, heads, dim)
    bits = torch.cat([bits, bits[:1]]).index_copy_(0, torch.where(real, slot, pool * page), code)[:-1]
    cache.view(torch.int8).copy_(bits.view(pool, page, heads, dim).permute(0, 2, 1, 3))
    scales.copy_(scale)
    return _gathered(cache, scales, s["every"], block, s["new_keys"].dtype), scales


def _round(x, cache):
    """The codes nearest to float64 values within the type's range, ties to even: rounded once, from 64 bits."""
    if cache == "int8":
        return x.round().to(torch.int8)
    least, digits = (-6, 3) if cache == "e4m3" else (-14, 2)
    step = _binade(x).clamp(min=2.0**least) * 2.0**-digits
    return ((x / step).round() * step).float().to(_CODE[cache])


def _binade(x):
    """The largest power of two that is not above |x|, of float64 values: their exponent bits (torch's powers are not exact)."""
    return (x.view(torch.int64) & 0x7FF0000000000000).view(torch.float64)


def _gathered(cache, scales, slots, block, dtype):
    page = cache.shape[2]
    slot = slots.long()
    x = cache[slot // page, :, slot % page].float() * scales[slot // page, :, slot % page // block][..., None]
    return x[:, 0::2].to(dtype), x[:, 1::2].to(dtype)


def _run_gather(s, case):
    if own:
        from ejkernel_amd.modules import quantized_cache_gather

        return quantized_cache_gather(s["cache"], s["scales"], s["slots"], dtype=_TYPE[case["dtype"]])
    return _gathered(s["cache"], s["scales"], s["slots"], case["block"], _TYPE[case["dtype"]])


def _run_tables(s, case):
    if own:
        from ejkernel_amd.modules import build_block_tables

        step = build_block_tables(s["new"], s["cached"], s["tables"], s["ring"], s["state"], s["count"], page_size=case["page"],
                                  total_tokens=s["tokens"])
        return (step.query_start_loc, step.context_lens, step.slot_mapping, step.positions, step.admitted, step.cached_lens,
                step.free_state, s["tables"], s["ring"])
    page, tokens = case["page"], s["tokens"]
    table, ring, cap = s["tables"], s["ring"], s["ring"].numel()
    new, cached = s["new"].long(), s["cached"].long()
    head, free = s["state"].long().unbind()
    have = (cached + page - 1) // page
    q = new.clamp(min=0)
    start = torch.cat([torch.zeros_like(q[:1]), q.cumsum(0)])
    fits = (cached + q <= table.shape[1] * page) & (start[1:] <= tokens)
    need = torch.where((q > 0) & fits, (cached + q + page - 1) // page - have, 0)
    taken = need.cumsum(0)
    admitted = (new >= 0) & fits & ((need == 0) | (taken <= free))
    got = torch.where(admitted, need, 0)
    back = torch.where(new < 0, have, 0)
    given = back.cumsum(0)
    ended = (new < 0) & (free + given <= cap)
    column = torch.arange(table.shape[1], device="cuda")
    fresh = (column >= have[:, None]) & (column < (have + got)[:, None])
    from_ring = ring[(head + (taken - need)[:, None] + column - have[:, None]) % cap]
    spot = torch.where((column < back[:, None]) & ended[:, None], (head + free + (given - back)[:, None] + column) % cap, cap)
    ring.copy_(torch.cat([ring, ring[:1]]).index_copy_(0, spot.view(-1), table.reshape(-1))[:-1])
    table.copy_(torch.where(fresh, from_ring, table))
    context = torch.where(admitted, cached + q, 0)
    kept = torch.where(admitted, cached + q, torch.where(ended, 0, cached))
    t = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(start[1:], t, right=True).clamp(max=q.numel() - 1)
    used = (t < start[-1]) & admitted[seq]
    pos = cached[seq] + t - start[seq]
    slot = table[seq, torch.where(used, pos // page, 0)].long() * page + pos % page
    state = torch.stack([(head + got.sum()) % cap, free - got.sum() + torch.where(ended, back, 0).sum()])
    whole = (start.clamp(max=tokens), context, torch.where(used, slot, -1), torch.where(used, pos, -1), admitted, kept, state)
    return tuple(x.int() for x in whole) + (table, ring)


# ------------------------------------------------------------------------------------------------ work and exact values


def work(case):
    if case["op"] == "attention":
        q, kv = _lengths(case)
        esize = 2 if case["dtype"] == "bf16" else 4
        w = case["window"] or 1 << 60
        first = np.maximum(kv - q - w + 1, 0)
        read = int((kv - first).sum())
        pairs = sum(int(np.minimum(np.arange(k - n, k) + 1, w).sum()) for n, k in zip(q.tolist(), kv.tolist()))
        heads, dim = 2 * case["kv_heads"], case["head_dim"]
        return {"bytes": read * heads * dim + -(-read // case["block"]) * heads * 4 + 2 * int(q.sum()) * case["q_heads"] * dim * esize + 4 * int((-(-kv // case["page"])).sum()),
                "flops": 4 * dim * case["q_heads"] * pairs}
    if case["op"] == "update":
        new, prior = _update_lengths(case)
        esize, row = (2 if case["dtype"] == "bf16" else 4), 2 * case["kv_heads"] * case["head_dim"]
        rows = int((-(-(prior % case["page"] + new) // case["page"])).sum() + 1) * case["page"]
        scales = 2 * case["kv_heads"] * 4 * (rows // case["block"])
        # the new rows in and their codes out; then every row of the pool in and its values out
        return {"bytes": int(new.sum()) * row * (esize + 1) + rows * row * (1 + esize) + 2 * scales, "flops": 2 * row * (int(new.sum()) + rows)}
    if case["op"] == "gather":
        esize, row = (2 if case["dtype"] == "bf16" else 4), 2 * case["kv_heads"] * case["head_dim"]
        return {"bytes": case["tokens"] * (row * (1 + esize) + 4) + -(-case["tokens"] // case["block"]) * 2 * case["kv_heads"] * 4, "flops": case["tokens"] * row}
    new, cached = _tables_lengths(case)
    page = case["page"]
    have = -(-cached // page)
    pages = int(np.where(new > 0, -(-(cached + new) // page) - have, have * (new < 0)).sum())
    tokens = int(np.maximum(new, 0).sum())
    # lengths in, five vectors out, each moved page in and out, a slot and a position for each token
    return {"bytes": 4 * (7 * case["seqs"] + 2 * pages + 2 * tokens), "flops": 8 * (case["seqs"] + tokens)}


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    block, page, cache, scales = case["block"], case["page"], s["cache"], s["scales"]
    if case["op"] == "gather":
        return _exact_rows(cache, scales, s["slots"], block)
    return _exact_attention(s, case) if case["op"] == "attention" else _exact_update(s, case)


def _exact_rows(cache, scales, slots, block):
    page = cache.shape[2]
    slot = slots.long()
    rows = cache.transpose(1, 2).reshape(-1, *cache[0, :, 0].shape)[slot].to(torch.float64)
    rows = rows * scales.transpose(1, 2).reshape(-1, scales.shape[1])[(slot // page) * scales.shape[2] + slot % page // block].double().unsqueeze(-1)
    return rows[:, 0::2], rows[:, 1::2]


def _exact_update(s, case):
    """Block by block of the step's tokens, in order, in 64 bits; a scale is held in 32 and rounded to them once."""
    cache, scales, block, page, qmax = s["cache"].clone(), s["scales"].clone(), case["block"], case["page"], _QMAX[case["cache"]]
    grid = _grid(case["cache"])
    heads, dim = cache.shape[1], cache.shape[3]
    new = torch.stack((s["new_keys"], s["new_values"]), dim=2).flatten(1, 2).double()
    slots = s["slots"].tolist()
    runs, t = [], 0
    while t < len(slots):
        n = 1
        while slots[t] >= 0 and t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % block:
            n += 1
        if slots[t] >= 0:
            runs.append((t, n))
        t += n
    if len(runs) > 6000:
        return None
    for t, n in runs:
        p, off = slots[t] // page, slots[t] % page
        b, inside = off // block, off % block
        rows = new[t:t + n].transpose(0, 1)
        peak = rows.abs().flatten(1).amax(1)
        want = torch.where(peak > 0, (peak / 127).clamp(min=2.0**-126), 0.0) if case["cache"] == "int8" else _power(peak, qmax)
        was = scales[p, :, b].double()
        now = torch.maximum(want.float().double(), was) if inside else want.float().double()
        if inside:
            at = slice(off - inside, off)
            redo = _nearest(cache[p, :, at].double() * was.view(-1, 1, 1) / now.clamp(min=1e-300).view(-1, 1, 1), grid)
            cache[p, :, at] = torch.where((now > was).view(-1, 1, 1), redo, cache[p, :, at].double()).to(torch.float32).to(cache.dtype)
        cache[p, :, off:off + n] = _nearest(rows / now.clamp(min=1e-300).view(-1, 1, 1), grid).to(torch.float32).to(cache.dtype)
        scales[p, :, b] = now.float()
    return _exact_rows(cache, scales, s["every"], block), scales.double()


def _power(peak, qmax):
    e = torch.ceil(torch.log2(peak.clamp(min=1e-300) / qmax) - 1e-9)  # a peak lies far further from a border than that
    e = torch.where(torch.exp2(e) * qmax < peak, e + 1, e).clamp(min=-126)
    return torch.where(peak > 0, torch.exp2(e), 0.0)


def _grid(cache):
    """Every value of the 8-bit type that is not negative, in order."""
    if cache == "int8":
        return torch.arange(128, dtype=torch.float64, device="cuda")
    codes = torch.arange(127 if cache == "e4m3" else 124, dtype=torch.uint8, device="cuda")
    return codes.view(_CODE[cache]).double()


def _nearest(x, grid):
    """The values of the grid nearest to x, a tie to the one of even place."""
    a = x.abs()
    hi = torch.searchsorted(grid, a.contiguous()).clamp(1, grid.numel() - 1)
    lo = hi - 1
    up, down = grid[hi] - a, a - grid[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.copysign(grid[pick], x)


def _exact_attention(s, case):
    q_lens, kv_lens = _lengths(case)
    if float(work(case)["flops"]) > 4e13:
        return None
    group, dim, page, block = case["q_heads"] // case["kv_heads"], case["head_dim"], case["page"], case["block"]
    out = torch.zeros(s["queries"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, m) in enumerate(zip(q_lens.tolist(), kv_lens.tolist())):
        key = torch.arange(m, device="cuda")
        slots = s["tables"][i].long()[key // page] * page + key % page
        k, v = _exact_rows(s["cache"][slots // page, :, slots % page].unsqueeze(2), s["scales"][slots // page, :, slots % page // block].unsqueeze(2), key, 1)
        pos = m - n + torch.arange(n, device="cuda")
        hide = key[None, :] > pos[:, None]
        if case["window"]:
            hide |= key[None, :] <= pos[:, None] - case["window"]
        for h in range(case["q_heads"]):
            z = s["queries"][at:at + n, h].double() @ k[:, h // group].T.contiguous() / math.sqrt(dim)
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            z[hide] = -math.inf
            if s["sinks"] is not None:
                z = torch.cat([z, s["sinks"][h].double().expand(n, -1)], dim=1)
            out[at:at + n, h] = torch.softmax(z, dim=1)[:, :m] @ v[:, h // group]
        at += n
    return out
