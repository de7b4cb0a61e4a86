"""quantized_cache_update and quantized_cache_gather on the GPU: codes and scales are those of the definition, bit for bit."""

import numpy as np
import pytest
import torch

from ejkernel_amd.modules import quantized_cache_gather, quantized_cache_update
from oracle import quantized_oracle as oracle
from tests.quantized_helpers import int32, random_cache, to_device

pytestmark = pytest.mark.gpu

KINDS = ("int8", "e4m3", "e5m2")


def rows(rng, tokens, heads, dim, dtype, spread=3.0):
    x = rng.standard_normal((tokens, heads, dim)) * np.exp(spread * rng.standard_normal((tokens, 1, 1)))
    t = torch.from_numpy(x.astype(np.float32))
    return t.to(torch.bfloat16) if dtype == "bf16" else t


def check_update(keys, values, codes, scales, slots, kind):
    cache, sc = to_device(codes, kind), torch.from_numpy(scales).to("cuda:0")
    got = quantized_cache_update(keys.to("cuda:0"), values.to("cuda:0"), cache, sc, int32(slots))
    torch.cuda.synchronize()
    assert got[0] is cache and got[1] is sc
    want, want_scales = oracle.cache_update(keys.double().numpy(), values.double().numpy(), codes, scales, list(slots), kind)
    np.testing.assert_array_equal(sc.cpu().numpy(), want_scales)
    np.testing.assert_array_equal(oracle.VALUES[kind][cache.view(torch.uint8).cpu().numpy()], oracle.VALUES[kind][want])
    return cache, sc


def runs(rng, pool, page, lengths, shuffle=True):
    """Slots of sequences of these lengths over distinct pages, each beginning somewhere in its first page."""
    order = list(rng.permutation(pool))
    out = []
    for n in lengths:
        at = int(rng.integers(0, page))
        pages = [order.pop() for _ in range(-(-(at + n) // page))]
        out += [pages[(at + i) // page] * page + (at + i) % page for i in range(n)]
    return np.array(out, np.int64)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,page,block", [(2, 128, 16, 16), (1, 64, 32, 8), (3, 96, 8, 4), (1, 256, 128, 64), (5, 16, 4, 4), (2, 240, 256, 256)])
def test_update(heads, dim, page, block, kind, dtype):
    rng = np.random.default_rng(dim + page)
    lengths = [1, 1, 3, page, 2 * page + 1, 1, 70, 129, 2, 1]
    pool = sum(n // page + 2 for n in lengths)
    slots = runs(rng, pool, page, lengths)
    slots = np.concatenate([slots[:5], [-1, -1, pool * page, 2**31 - 1, -(2**31)], slots[5:], [-1]])
    codes, scales = random_cache(rng, pool, 2 * heads, page, dim, block, kind)
    check_update(rows(rng, len(slots), heads, dim, dtype), rows(rng, len(slots), heads, dim, dtype), codes, scales, slots, kind)


@pytest.mark.parametrize("kind", KINDS)
def test_token_by_token_history(kind):
    """A sequence written a token at a time: every step's scale and codes follow from the last step's."""
    rng = np.random.default_rng(7)
    codes, scales = random_cache(rng, 4, 4, 16, 64, 8, kind)
    for step in range(40):
        k, v = rows(rng, 2, 2, 64, "bf16", 1.0), rows(rng, 2, 2, 64, "bf16", 1.0)
        cache, sc = check_update(k, v, codes, scales, [2 * 16 + step % 16 if step < 16 else 16 + step % 16, (step * 3) % 16 if step % 5 else -1], kind)
        codes, scales = cache.view(torch.uint8).cpu().numpy(), sc.cpu().numpy()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kind", KINDS)
def test_values_at_the_edges(kind, dtype):
    """Zeros, the least and the largest numbers, infinities, NaN, ties, old scales of zero and of no number."""
    rng = np.random.default_rng(8)
    codes, scales = random_cache(rng, 12, 2, 8, 64, 8, kind)
    x = torch.zeros((24, 1, 64))
    x[1] = 1e-40
    x[2, 0, 0], x[2, 0, 1] = 3e38, 1.0
    x[3, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 2.0])
    x[4] = float("nan")
    x[5] = float("inf")
    x[6, 0] = torch.arange(64).float() - 31.5      # with 127 in the row: halves between int8 codes
    x[6, 0, 0] = 127.0
    x[7, 0] = torch.linspace(-448, 448, 64)
    x[8:] = torch.from_numpy(rng.standard_normal((16, 1, 64)).astype(np.float32))
    x[9] *= 2.0**-140
    x[10, 0, 0] = 448.0
    x[11, 0, 0] = 449.0
    x[12, 0, 0] = 57344.0
    x[13, 0, 0] = 57600.0
    x = x.to(torch.bfloat16) if dtype == "bf16" else x
    slots = list(range(0, 64, 8)) + [64, 65, 66, 67, 72 + 1, 72 + 2, 80 + 3, 88 + 7] + [-1] * 8
    scales[9, 0], scales[9, 1], scales[10, 0], scales[10, 1] = 0.0, -1.0, np.nan, 2.0**-126
    cache, sc = to_device(codes, kind), torch.from_numpy(scales.copy()).to("cuda:0")
    quantized_cache_update(x.to("cuda:0"), x.to("cuda:0"), cache, sc, int32(slots))
    torch.cuda.synchronize()
    sane = scales.copy()
    sane[~(sane > 0)] = 0  # an old scale that is no positive number counts as none
    want, want_scales = oracle.cache_update(x.double().numpy(), x.double().numpy(), codes, sane, slots, kind)
    touched = sorted({s // 8 for s in slots if s >= 0})
    np.testing.assert_array_equal(sc.cpu().numpy()[touched], want_scales[touched])
    np.testing.assert_array_equal(oracle.VALUES[kind][cache.view(torch.uint8).cpu().numpy()], oracle.VALUES[kind][want])
    k, v = quantized_cache_gather(cache, sc, int32([s for s in slots if s >= 0]))
    assert torch.isfinite(k).all() and torch.isfinite(v).all()


def test_ties_are_decided_on_the_exact_quotient():
    """int8 codes of rows of which many lie within an ulp of the middle between two codes."""
    rng = np.random.default_rng(9)
    a = rng.uniform(0.5, 2.0, size=(400, 1)).astype(np.float32)
    s = (a / np.float32(127)).astype(np.float32)
    x = (rng.integers(-126, 126, size=(400, 64)) + 0.5).astype(np.float32) * s
    x = np.nextafter(x, np.where(rng.integers(0, 3, size=x.shape) == 0, np.float32(9), np.where(rng.integers(0, 2, size=x.shape) == 0, x, np.float32(-9)))).astype(np.float32)
    x[:, 0] = a[:, 0]
    x = torch.from_numpy(x)[:, None]
    codes, scales = random_cache(rng, 100, 2, 16, 64, 4, "int8")
    check_update(x, -x, codes, scales, [4 * t for t in range(400)], "int8")


def test_rows_come_from_strided_views():
    rng = np.random.default_rng(10)
    codes, scales = random_cache(rng, 8, 4, 16, 128, 16, "e4m3")
    slots = list(range(5, 100))
    fused = rows(rng, 95, 10, 128, "bf16").to("cuda:0")
    keys, values = fused[:, 6:8], fused[:, 8:10]
    want = check_update(keys.cpu(), values.cpu(), codes, scales, slots, "e4m3")
    odd = torch.empty(95 * 256 + 1, dtype=torch.bfloat16, device="cuda:0")[1:].view(95, 2, 128)
    odd.copy_(values)
    for k, v in ((keys, values), (keys.transpose(0, 1).contiguous().transpose(0, 1), values), (keys, odd),
                 (torch.cat([keys, keys], 2)[..., ::2].clone(), values)):
        if not torch.equal(k, keys):
            continue
        cache, sc = to_device(codes, "e4m3"), torch.from_numpy(scales).to("cuda:0")
        quantized_cache_update(k, v, cache, sc, int32(slots))
        assert torch.equal(cache.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(sc, want[1])
    one = keys[:, :1].expand(-1, 2, -1)  # one head's keys for both: stride 0
    check_update(one.cpu(), values.cpu(), codes, scales, slots, "e4m3")
    cache, sc = to_device(codes, "e4m3"), torch.from_numpy(scales).to("cuda:0")
    quantized_cache_update(one, values, cache, sc, int32(slots))
    ref, ref_sc = oracle.cache_update(one.double().cpu().numpy(), values.double().cpu().numpy(), codes, scales, slots, "e4m3")
    np.testing.assert_array_equal(sc.cpu().numpy(), ref_sc)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 2, 63, 300])
def test_gather(tokens, kind, dtype):
    rng = np.random.default_rng(tokens)
    for heads, dim, page, block in ((2, 128, 16, 4), (1, 80, 64, 64), (3, 256, 8, 8)):
        codes, scales = random_cache(rng, 9, 2 * heads, page, dim, block, kind)
        slots = rng.integers(-2, 9 * page + 2, size=tokens)  # repeated ones, and some outside
        k, v = quantized_cache_gather(to_device(codes, kind), torch.from_numpy(scales).to("cuda:0"), int32(slots), dtype=dtype)
        wk, wv = oracle.cache_gather(codes, scales, list(slots), kind)
        for got, want in ((k, wk), (v, wv)):
            # code * scale in float32, then to the type: both round to nearest, and a bf16 code times a scale has 32 bits
            as32 = torch.from_numpy(want.astype(np.float32))
            assert got.dtype == dtype and torch.equal(got.cpu(), as32.to(dtype))


def test_empty_calls():
    codes, scales = random_cache(np.random.default_rng(1), 2, 2, 16, 64, 16, "int8")
    cache, sc = to_device(codes, "int8"), torch.from_numpy(scales).to("cuda:0")
    none = torch.empty((0, 1, 64), dtype=torch.bfloat16, device="cuda:0")
    quantized_cache_update(none, none, cache, sc, int32([]))
    k, v = quantized_cache_gather(cache, sc, int32([]))
    assert k.shape == v.shape == (0, 1, 64) and np.array_equal(cache.view(torch.uint8).cpu().numpy(), codes)


def test_update_in_a_graph_follows_its_slots():
    rng = np.random.default_rng(11)
    codes, scales = random_cache(rng, 6, 4, 16, 128, 16, "int8")
    cache, sc = to_device(codes, "int8"), torch.from_numpy(scales).to("cuda:0")
    k, v, slots = rows(rng, 3, 2, 128, "bf16").to("cuda:0"), rows(rng, 3, 2, 128, "bf16").to("cuda:0"), int32([0, 20, -1])
    quantized_cache_update(k, v, cache, sc, int32([-1, -1, -1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        quantized_cache_update(k, v, cache, sc, slots)
        back = quantized_cache_gather(cache, sc, slots)
    for step in range(5):
        s = [step, 20 + step, -1 if step % 2 else 64 + step]
        x, y = rows(rng, 3, 2, 128, "bf16"), rows(rng, 3, 2, 128, "bf16")
        k.copy_(x), v.copy_(y), slots.copy_(int32(s))
        graph.replay()
        torch.cuda.synchronize()
        codes, scales = oracle.cache_update(x.double().numpy(), y.double().numpy(), codes, scales, s, "int8")
        np.testing.assert_array_equal(cache.view(torch.uint8).cpu().numpy(), codes)
        np.testing.assert_array_equal(sc.cpu().numpy(), scales)
        wk, _ = oracle.cache_gather(codes, scales, s, "int8")
        assert torch.equal(back[0].cpu(), torch.from_numpy(wk.astype(np.float32)).to(torch.bfloat16))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim", [(1, 16), (3, 48), (2, 128), (2, 256)])
def test_single_tokens_beside_runs(heads, dim, kind):
    """Single tokens alone, with holes, and in front of a run that begins at the last token of 64 or goes on behind them."""
    rng = np.random.default_rng(dim)
    page, block = 32, 8
    single = lambda n, first: [(first + i) * page + int(rng.integers(0, page)) for i in range(n)]  # noqa: E731
    for slots in (single(64, 0), single(130, 0), single(40, 0) + [-1] * 30 + single(9, 40), single(63, 0) + [70 * page + 3 + i for i in range(12)],
                  single(63, 0) + [70 * page + 7, 70 * page + 8] + single(5, 90), single(64, 0) + [80 * page + i for i in range(70)],
                  [5 * page + 30 + i for i in range(2)] + [6 * page], [-1] * 64 + single(3, 0), [9 * page + 31]):
        codes, scales = random_cache(rng, 150, 2 * heads, page, dim, block, kind)
        keys, values = rows(rng, len(slots), heads, dim, "bf16"), rows(rng, len(slots), heads, dim, "bf16")
        keys[:: 7, :, 1::2] = float("inf")
        values[2:: 9, 0, 0] = float("nan")
        check_update(keys, values, codes, scales, slots, kind)


def test_a_pool_beyond_four_gigabytes():
    """Codes and scales beyond 2**32 bytes: the same rows as in a small pool, written, read and attended to."""
    from ejkernel_amd.modules import quantized_ragged_page_attention

    rng = np.random.default_rng(1)
    heads, dim, page, block, lengths = 8, 128, 16, 4, [100, 37]
    need = sum(-(-n // page) for n in lengths)
    keys, values = rows(rng, sum(lengths), heads, dim, "bf16", 0.5).to("cuda:0"), rows(rng, sum(lengths), heads, dim, "bf16", 0.5).to("cuda:0")
    queries = rows(rng, 41, 16, dim, "bf16", 0.1).to("cuda:0")
    results = []
    for pool, last in ((need, False), ((9 << 29) // (2 * heads * page * dim), True)):
        cache = torch.zeros((pool, 2 * heads, page, dim), dtype=torch.int8, device="cuda:0")
        scales = torch.zeros((pool, 2 * heads, page // block), device="cuda:0")
        pages = list(range(pool - need, pool)) if last else list(range(need))
        table = np.full((2, 7), -1)
        slots, at = [], 0
        for s, n in enumerate(lengths):
            count = -(-n // page)
            table[s, :count] = pages[at: at + count]
            slots += [int(table[s, i // page]) * page + i % page for i in range(n)]
            at += count
        assert not last or min(slots) * 2 * heads * dim > 2**32
        quantized_cache_update(keys, values, cache, scales, int32(slots))
        out = quantized_ragged_page_attention(queries, cache, scales, int32(lengths), int32(table), int32([0, 40, 41]), int32([2]))
        results.append((*quantized_cache_gather(cache, scales, int32(slots)), out))
        assert torch.isfinite(out).all() and out.abs().amax(-1).min() > 0
        assert not last or not cache[: pool - need].any()
    for a, b in zip(*results):
        assert torch.equal(a, b)
