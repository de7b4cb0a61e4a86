"""Plain restatements, in float64 and Python integers, of the operations on the 8-bit cache with block scales.

They follow the definitions in ``include/rpa_mi355x.h`` one token, one block and one request at a time and share
nothing with the kernels.  Codes are numpy arrays of uint8 (the bytes of the cache); scales are float32.
"""

from __future__ import annotations

import math

import numpy as np

QMAX = {"int8": 127.0, "e4m3": 448.0, "e5m2": 57344.0}


def _float8_values(exponent_bits: int, mantissa_bits: int) -> np.ndarray:
    bias = 2 ** (exponent_bits - 1) - 1
    v = np.zeros(256)
    for b in range(256):
        e, m = (b & 127) >> mantissa_bits, b & (2**mantissa_bits - 1)
        x = m * 2.0 ** (1 - bias - mantissa_bits) if e == 0 else (1 + m / 2**mantissa_bits) * 2.0 ** (e - bias)
        if exponent_bits == 5 and e == 31:
            x = math.inf if m == 0 else math.nan
        if exponent_bits == 4 and b & 127 == 127:
            x = math.nan
        v[b] = -x if b & 128 else x
    return v


VALUES = {"int8": np.arange(256).astype(np.uint8).view(np.int8).astype(np.float64), "e4m3": _float8_values(4, 3),
          "e5m2": _float8_values(5, 2)}


def nearest_codes(x: np.ndarray, kind: str) -> np.ndarray:
    """Bytes of the codes nearest to x (within the type's range), ties to even."""
    if kind == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    top = {"e4m3": 0x7E, "e5m2": 0x7B}[kind]
    grid = VALUES[kind][: top + 1]
    a = np.abs(x)
    hi = np.clip(np.searchsorted(grid, a), 1, top)
    up, down = grid[hi] - a, a - grid[hi - 1]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1).astype(np.uint8)
    return code | (np.signbit(x).astype(np.uint8) << 7)


def fresh_scale(a: float, kind: str) -> np.float32:
    if a == 0:
        return np.float32(0)
    if kind == "int8":
        return np.maximum(np.float32(a) / np.float32(127), np.float32(2.0**-126))
    e = -126
    while QMAX[kind] * 2.0**e < a:
        e += 1
    return np.float32(2.0**e)


def cache_update(keys, values, codes, scales, slots, kind):
    """New ``(codes, scales)``; keys / values float64 ``[T, Hkv, D]``, codes uint8 ``[P, 2 Hkv, page, D]``."""
    codes, scales = codes.copy(), scales.copy()
    pages, heads, page, _ = codes.shape
    block = page // scales.shape[2]
    ok = [0 <= s < pages * page for s in slots]
    t = 0
    while t < len(slots):
        if not ok[t]:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % block:
            n += 1
        p, off = slots[t] // page, slots[t] % page
        b, inside = off // block, off % block
        for h in range(heads):
            x = (values if h % 2 else keys)[t:t + n, h // 2].astype(np.float64)
            finite = np.isfinite(x)
            s = fresh_scale(float(np.abs(x[finite]).max(initial=0.0)), kind)
            old = scales[p, h, b]
            if inside and old > s:
                s = old
            if inside and s > old:
                row = codes[p, h, off - inside:off]
                codes[p, h, off - inside:off] = nearest_codes(VALUES[kind][row] * float(old) / float(s), kind)
            if s == 0:
                codes[p, h, off:off + n] = 0
            else:
                y = np.where(np.isnan(x), 0.0, np.clip(np.where(np.isnan(x), 0.0, x) / float(s), -QMAX[kind], QMAX[kind]))
                codes[p, h, off:off + n] = nearest_codes(y, kind)
            scales[p, h, b] = s
        t += n
    return codes, scales


def cache_values(codes, scales, kind):
    """Float64 values of the whole pool, ``[P, 2 Hkv, page, D]``."""
    block = codes.shape[2] // scales.shape[2]
    return VALUES[kind][codes] * np.repeat(scales.astype(np.float64), block, axis=2)[..., None]


def cache_gather(codes, scales, slots, kind):
    v = cache_values(codes, scales, kind)
    pages, heads, page, dim = v.shape
    out = np.zeros((len(slots), heads, dim))
    for t, s in enumerate(slots):
        if 0 <= s < pages * page:
            out[t] = v[s // page, :, s % page]
    return out[:, 0::2], out[:, 1::2]


def attention(queries, codes, scales, lens, tables, starts, num_seqs, kind, *, sinks=None, scale=None, cap=None, window=None):
    """``(out, size, reach)`` in float64: the output, the same sum over |v| (what errors of the probabilities are relative
    to), and per row the largest sum of |q k| * scale over its keys (what errors of the logits are relative to).  Masked
    keys are left out of the sums, so what lies there does not matter."""
    dim = queries.shape[2]
    scale = dim**-0.5 if scale is None else scale
    out, size, reach = np.zeros(queries.shape), np.zeros(queries.shape), np.zeros(queries.shape[:2])
    pages, heads, page, _ = codes.shape
    block = page // scales.shape[2]
    group = queries.shape[1] // (heads // 2)
    for s in range(num_seqs):
        q0, q1, m = starts[s], starts[s + 1], lens[s]
        key = np.arange(m)
        pg, off = np.clip(tables[s][key // page], 0, pages - 1), key % page
        with np.errstate(invalid="ignore"):
            rows = VALUES[kind][codes[pg, :, off]] * scales[pg, :, off // block].astype(np.float64)[..., None]
        for t in range(q0, q1):
            pos = m - (q1 - q0) + t - q0
            seen = key <= pos
            if window is not None:
                seen &= key > pos - window
            if not seen.any():
                continue
            for h in range(queries.shape[1]):
                x = rows[seen, 2 * (h // group)] @ queries[t, h].astype(np.float64) * scale
                if cap is not None:
                    x = cap * np.tanh(x / cap)
                extra = np.zeros(0) if sinks is None else sinks[h].astype(np.float64)
                top = max(x.max(), extra.max(initial=-np.inf))
                p = np.exp(x - top)
                p /= p.sum() + np.exp(extra - top).sum()
                v = rows[seen, 2 * (h // group) + 1]
                out[t, h], size[t, h] = p @ v, p @ np.abs(v)
                reach[t, h] = (np.abs(rows[seen, 2 * (h // group)]) @ np.abs(queries[t, h].astype(np.float64))).max() * abs(scale)
    return out, size, reach


def block_tables(query_lens, cached_lens, tables, ring, state, num_seqs, page, total):
    """Every result of the step as Python / numpy integers: a dict that also holds the new tables and ring."""
    tables, ring = tables.copy(), ring.copy()
    n_all, columns = tables.shape
    cap = len(ring)
    head, count = int(state[0]) % cap, min(max(int(state[1]), 0), cap)
    r = {"query_start_loc": [0], "context_lens": [], "slot_mapping": [-1] * total, "positions": [-1] * total, "admitted": [],
         "cached_lens": []}
    at = need_sum = back_sum = took = gave = 0
    for s in range(n_all):
        q = int(query_lens[s]) if s < num_seqs else 0
        cached = min(max(int(cached_lens[s]), 0), columns * page) if s < num_seqs else 0
        have, end = -(-cached // page), at + max(q, 0)
        context, admitted, kept = 0, 0, cached
        if q == 0:
            context, admitted = cached, 1
        elif q > 0 and cached + q <= columns * page and end <= total:
            need = -(-(cached + q) // page) - have
            if need == 0 or need_sum + need <= count:
                for k in range(need):
                    tables[s, have + k] = ring[(head + need_sum + k) % cap]
                took += need
                context, admitted, kept = cached + q, 1, cached + q
                for i in range(q):
                    pos = cached + i
                    r["positions"][at + i] = pos
                    r["slot_mapping"][at + i] = int(tables[s, pos // page]) * page + pos % page
            need_sum += need
        elif q < 0:
            if count + back_sum + have <= cap:
                for k in range(have):
                    ring[(head + count + back_sum + k) % cap] = tables[s, k]
                gave += have
                kept = 0
            back_sum += have
        at = end
        r["query_start_loc"].append(min(at, total))
        r["context_lens"].append(context)
        r["admitted"].append(admitted)
        r["cached_lens"].append(kept if s < num_seqs else int(cached_lens[s]))
    r["free_state"] = [(head + took) % cap, count - took + gave]
    return r | {"tables": tables, "ring": ring}
