"""Batches over the 8-bit cache with block scales, and the bounds their results are held to."""

import numpy as np
import torch

from oracle import quantized_oracle as oracle

TORCH_KIND = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
POISON = {"int8": 0x80, "e4m3": 0x7F, "e5m2": 0x7D}  # a code that no update writes; NaN in the floating types


def to_device(codes, kind, device="cuda:0"):
    return torch.from_numpy(codes.copy()).to(device).view(TORCH_KIND[kind])


def int32(x, device="cuda:0"):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


def random_cache(rng, pages, heads, page, dim, block, kind):
    """Finite codes of every size and scales of a spread of 2**6."""
    if kind == "int8":
        codes = rng.integers(-127, 128, size=(pages, heads, page, dim)).astype(np.int8).view(np.uint8)
        scales = np.exp2(rng.uniform(-8, -5, size=(pages, heads, page // block)))
    else:
        codes = oracle.nearest_codes(np.clip(rng.standard_normal((pages, heads, page, dim)), -4, 4) * (oracle.QMAX[kind] / 4), kind)
        scales = np.exp2(np.floor(rng.uniform(-2, 2, size=(pages, heads, page // block)))) / (oracle.QMAX[kind] / 4)
    return codes, scales.astype(np.float32)


class Batch:
    """Sequences (new tokens, keys) over a scattered pool.  What no row may read is poisoned: pages nobody owns, rows and
    scales behind a sequence's last key and in front of its first visible one, table entries behind its pages."""

    def __init__(self, seqs, *, q_heads, kv_heads, dim, page, block, kind, dtype="bf16", window=None, cap=None, sinks=0, scale=None,
                 slack=0, spare_seqs=0, seed=0):
        rng = np.random.Generator(np.random.PCG64(seed))
        self.kind, self.dtype, self.window, self.cap, self.scale = kind, dtype, window, cap, scale
        q, kv = np.array([a for a, _ in seqs], np.int64), np.array([b for _, b in seqs], np.int64)
        counts = -(-kv // page)
        columns = int(counts.max(initial=0)) + 2
        pool = int(counts.sum()) + 3
        self.codes, self.scales = random_cache(rng, pool, 2 * kv_heads, page, dim, block, kind)
        self.tables = rng.choice([-7, pool + 5, 1 << 30], size=(len(seqs) + spare_seqs, columns)).astype(np.int64)
        order = rng.permutation(pool)
        used = np.zeros((pool, page), bool)
        at = 0
        for s, (n, m) in enumerate(seqs):
            self.tables[s, : counts[s]] = order[at: at + counts[s]]
            at += counts[s]
            first = max(m - n - window + 1, 0) if window else 0
            key = np.arange(first, m)
            used[self.tables[s, key // page], key % page] = True
        at_block = used.reshape(pool, page // block, block).any(2)
        self.codes[np.broadcast_to(~used[:, None, :, None], self.codes.shape)] = POISON[kind]
        self.scales[np.broadcast_to(~at_block[:, None], self.scales.shape)] = np.nan
        self.lens = np.concatenate([kv, np.full(spare_seqs, 999)])
        self.starts = np.concatenate([[0], np.cumsum(q), np.full(spare_seqs, 10**6)])
        self.num_seqs = len(seqs)
        x = torch.from_numpy(rng.standard_normal((int(q.sum()) + slack, q_heads, dim)).astype(np.float32))
        self.queries = x.to(torch.bfloat16) if dtype == "bf16" else x
        self.sinks = rng.standard_normal((q_heads, sinks)).astype(np.float32) if sinks else None
        self.rows = int(q.sum())

    def args(self, device="cuda:0"):
        sinks = () if self.sinks is None else (torch.from_numpy(self.sinks).to(device),)
        return (self.queries.to(device), to_device(self.codes, self.kind, device), torch.from_numpy(self.scales).to(device),
                int32(self.lens, device), int32(self.tables, device), int32(self.starts, device), int32([self.num_seqs], device), *sinks)

    def kwargs(self):
        return dict(logits_soft_cap=self.cap, sliding_window=self.window, softmax_scale=self.scale)

    def check(self, out):
        check_attention(out, self.queries, self.codes, self.scales, self.lens, self.tables, self.starts, self.num_seqs, self.kind,
                        sinks=self.sinks, scale=self.scale, cap=self.cap, window=self.window)


def check_attention(out, queries, codes, scales, lens, tables, starts, num_seqs, kind, **kw):
    """Holds an output to the float64 evaluation.

    The logits are sums of dim products in fp32 with a handful of roundings behind them: off by (dim + 16) 2**-24 of the
    sum of magnitudes at most (``reach``; the cap only shrinks that), and a probability by that, twice (its sum).  The sum
    of n fp32 terms adds n 2**-24 twice, the exponential and the joining of parts a few units.  With bf16 queries each
    probability times value scale is rounded once (2**-8 of it: 2**-8 of ``size`` in all) and the result once.  A probability
    below 2**-126 of its row's largest is no normal fp32 number and may vanish, which n of them do to the sum by n 2**-126
    of the largest value at most.
    """
    x = queries.float().numpy()
    with np.errstate(invalid="ignore"):
        values = np.abs(oracle.cache_values(codes, scales, kind)[:, 1::2])
    want, size, reach = oracle.attention(x, codes, scales, lens, tables, starts, num_seqs, kind, **kw)
    got = out.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    logit = (x.shape[2] + 16) * 2.0**-24 * reach[..., None]
    bound = size * (2 * logit + (2 * np.max(lens[:num_seqs], initial=0) + 64) * 2.0**-24) + 1e-37
    bound = bound + np.max(lens[:num_seqs], initial=0) * 2.0**-126 * values[np.isfinite(values)].max(initial=0.0)
    if queries.dtype == torch.bfloat16:
        bound = bound + 2.0**-8 * (1 + 2.0**-7) * (size + np.abs(want))
    else:
        bound = bound + 2.0**-24 * np.abs(want)
    worst = (np.abs(got - want) - bound).max(initial=-1.0)
    assert worst <= 0, f"off by {np.abs(got - want).max():.3g}, {worst:.3g} over the bound"
    assert not got[starts[num_seqs]:].any(), "rows behind the last sequence must be zeros"
