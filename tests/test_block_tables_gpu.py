"""build_block_tables on the GPU against a request-by-request restatement, and the serving step it begins."""

import numpy as np
import pytest
import torch

from ejkernel_amd.modules import build_block_tables, quantized_cache_gather, quantized_cache_update, quantized_ragged_page_attention
from oracle import quantized_oracle as oracle
from tests.quantized_helpers import check_attention, int32, random_cache, to_device

pytestmark = pytest.mark.gpu


def scene(rng, n, page, context, chunk, *, spare, extra_columns=1, ended=0.1, idle=0.1, pool_extra=0):
    cached = rng.integers(0, context + 1, size=n)
    q = np.where(rng.random(n) < 0.3, rng.integers(1, chunk + 1, size=n), 1)
    q[rng.random(n) < idle] = 0
    q[rng.random(n) < ended] = -rng.integers(1, 5)
    have = -(-cached // page)
    columns = -(-(context + chunk) // page) + extra_columns - 1
    ids = rng.permutation(int(have.sum()) + spare + pool_extra)
    tables = np.full((n, columns), -1, np.int64)
    tables[np.arange(columns)[None] < have[:, None]] = ids[: have.sum()]
    ring = np.full(len(ids), -9, np.int64)
    head = int(rng.integers(0, len(ids)))
    ring[(head + np.arange(spare)) % len(ids)] = ids[have.sum(): have.sum() + spare]
    return q, cached, tables, ring, [head, spare]


def check(q, cached, tables, ring, state, num_seqs, page, total):
    t, r = int32(tables), int32(ring)
    q_t, c_t, s_t = int32(q), int32(cached), int32(state)
    got = build_block_tables(q_t, c_t, t, r, s_t, int32([num_seqs]), page_size=page, total_tokens=total)
    torch.cuda.synchronize()
    want = oracle.block_tables(q, cached, np.asarray(tables), np.asarray(ring), state, min(max(num_seqs, 0), len(q)), page, total)
    for name in got._fields:
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), want[name], err_msg=name)
    np.testing.assert_array_equal(t.cpu().numpy(), want["tables"])
    np.testing.assert_array_equal(r.cpu().numpy(), want["ring"])
    assert np.array_equal(q_t.cpu().numpy(), q) and np.array_equal(c_t.cpu().numpy(), cached) and np.array_equal(s_t.cpu().numpy(), state)
    return got


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 256, 1000, 1024, 1025, 3000])
@pytest.mark.parametrize("page", [1, 4, 16, 48])
def test_steps(n, page):
    rng = np.random.default_rng(n + page)
    for spare in (0, n // 3 + 1, 40 * n):
        q, cached, tables, ring, state = scene(rng, n, page, 200, 70, spare=spare)
        total = int(np.maximum(q, 0).sum())
        check(q, cached, tables, ring, state, n, page, total + 7)


@pytest.mark.parametrize("total_of", [lambda s: 0, lambda s: s // 2, lambda s: s, lambda s: s + 5000])
@pytest.mark.parametrize("count_of", [lambda n: 0, lambda n: n // 2, lambda n: n, lambda n: n + 9, lambda n: -3])
def test_static_shapes_larger_and_smaller_than_the_batch(total_of, count_of):
    rng = np.random.default_rng(5)
    for n in (5, 40, 1500):
        q, cached, tables, ring, state = scene(rng, n, 8, 100, 30, spare=3 * n)
        check(q, cached, tables, ring, state, count_of(n), 8, total_of(int(np.maximum(q, 0).sum())))


def test_requests_at_the_limits():
    tables, ring = np.arange(12).reshape(3, 4), np.arange(100, 120)
    for q, cached in (([1, 16, 17], [63, 48, 48]), ([64, 65, 1], [0, 0, 64]), ([2**31 - 1, 1, 2**31 - 1], [5, 16, 64]), ([-1, -1, -1], [64, 1, 0]),
                      ([1, 1, 1], [-5, 10**9, 16]), ([0, 0, 0], [64, 3, 0])):
        for state in ([0, 20], [19, 3], [-1, 5], [45, 99], [3, -2], [0, 0]):
            check(np.array(q), np.array(cached), tables, ring, state, 3, 16, 90)


def test_a_ring_that_cannot_hold_what_comes_back_keeps_the_request():
    tables, ring = np.arange(40).reshape(5, 8), np.arange(50, 60)
    check(np.array([-1, 3, -1, -1, 40]), np.array([33, 16, 64, 20, 10]), tables, ring, [7, 4], 5, 16, 100)


def test_the_same_call_twice_gives_the_same():
    """The inputs that name a step are left alone, so the step can be taken again."""
    rng = np.random.default_rng(6)
    q, cached, tables, ring, state = scene(rng, 300, 16, 500, 40, spare=500)
    t, r, args = int32(tables), int32(ring), (int32(q), int32(cached))
    first = build_block_tables(*args, t, r, int32(state), 300, page_size=16, total_tokens=5000)
    tables_1, ring_1 = t.clone(), r.clone()
    second = build_block_tables(*args, t, r, int32(state), 300, page_size=16, total_tokens=5000)
    assert all(torch.equal(a, b) for a, b in zip(first, second)) and torch.equal(t, tables_1) and torch.equal(r, ring_1)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_serving_steps(kind, captured):
    """Requests that arrive, grow, are refused, end and come back: tables -> update -> attention, eager and as one graph.

    The attention is held to the float64 evaluation over the cache that the update left, that cache to the definition bit
    for bit, and the rows of the step itself to what was written: within half a step of their int8 scale."""
    rng = np.random.default_rng(12)
    n, page, block, heads, group, dim, pool, columns, total = 5, 16, 8, 2, 4, 64, 14, 6, 64
    codes, scales = random_cache(rng, pool, 2 * heads, page, dim, block, kind)
    cache, sc = to_device(codes, kind), torch.from_numpy(scales).to("cuda:0")
    tables, ring = int32(np.full((n, columns), -1)), int32(rng.permutation(pool))
    q_lens, cached, state, count = int32(np.zeros(n)), int32(np.zeros(n)), int32([0, pool]), int32([n])
    x = torch.zeros((total, heads * (group + 2), dim), dtype=torch.bfloat16, device="cuda:0")

    def step():
        s = build_block_tables(q_lens, cached, tables, ring, state, count, page_size=page, total_tokens=total)
        quantized_cache_update(x[:, heads * group: heads * (group + 1)], x[:, heads * (group + 1):], cache, sc, s.slot_mapping)
        out = quantized_ragged_page_attention(x[:, : heads * group], cache, sc, s.context_lens, tables, s.query_start_loc, count)
        rows = quantized_cache_gather(cache, sc, s.slot_mapping, dtype=torch.float32)
        cached.copy_(s.cached_lens), state.copy_(s.free_state)
        return s, out, rows

    if captured:
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                results = step()
        torch.cuda.synchronize()
    ref = dict(tables=np.full((n, columns), -1), ring=ring.cpu().numpy().astype(np.int64), cached=np.zeros(n, np.int64), state=[0, pool])
    ref["codes"], ref["scales"] = codes, scales
    plan = [[20, 1, 0, 0, 0], [1, 40, 3, 0, 0], [1, 1, 1, 60, 0], [1, 1, 1, 1, 5], [1, -1, 1, 17, 1], [2, 33, 1, 1, 1], [-1, 1, -1, 1, 30], [64, 0, 0, 0, 0], [1, 1, 1, 1, 1]]
    refused = 0
    for q in plan:
        q_lens.copy_(int32(q))
        x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
        if captured:
            graph.replay()
        else:
            results = step()
        torch.cuda.synchronize()
        s, out, rows = results
        want = oracle.block_tables(q, ref["cached"], ref["tables"], ref["ring"], ref["state"], n, page, total)
        for name in s._fields:
            np.testing.assert_array_equal(getattr(s, name).cpu().numpy(), want[name], err_msg=name)
        np.testing.assert_array_equal(tables.cpu().numpy(), want["tables"])
        np.testing.assert_array_equal(ring.cpu().numpy(), want["ring"])
        refused += sum(a == 0 and n_new > 0 for a, n_new in zip(want["admitted"], q))
        h = x.double().cpu().numpy()
        k, v = h[:, heads * group: heads * (group + 1)], h[:, heads * (group + 1):]
        ref["codes"], ref["scales"] = oracle.cache_update(k, v, ref["codes"], ref["scales"], want["slot_mapping"], kind)
        np.testing.assert_array_equal(sc.cpu().numpy(), ref["scales"])
        np.testing.assert_array_equal(oracle.VALUES[kind][cache.view(torch.uint8).cpu().numpy()], oracle.VALUES[kind][ref["codes"]])
        wk, wv = oracle.cache_gather(ref["codes"], ref["scales"], want["slot_mapping"], kind)
        assert np.array_equal(rows[0].cpu().numpy(), wk.astype(np.float32)) and np.array_equal(rows[1].cpu().numpy(), wv.astype(np.float32))
        if kind == "int8":
            for t, slot in enumerate(want["slot_mapping"]):
                if slot >= 0:
                    for got, new, first in ((wk, k, 0), (wv, v, 1)):
                        half = ref["scales"][slot // page, first::2, slot % page // block].astype(np.float64)[:, None] / 2
                        assert (np.abs(got[t] - new[t]) <= half * (1 + 1e-12)).all()
        starts = np.array(want["query_start_loc"])
        check_attention(out, x[:, : heads * group].cpu(), ref["codes"], ref["scales"], np.array(want["context_lens"]), want["tables"], starts, n, kind)
        ref.update(tables=want["tables"], ring=want["ring"], cached=np.array(want["cached_lens"]), state=want["free_state"])
    assert refused, "the plan is meant to run out of pages at least once"


@pytest.mark.parametrize("n", [1025, 2048, 4096, 4097, 9000])
@pytest.mark.parametrize("idle", [slice(0, 700), slice(100, 1000), slice(300, None)])
def test_many_requests_with_long_idle_stretches(n, idle):
    """Tokens whose request lies far behind the previous token's, and requests of several threads' share."""
    rng = np.random.default_rng(n)
    q, cached, tables, ring, state = scene(rng, n, 16, 100, 40, spare=2 * n)
    q[idle] = 0
    check(q, cached, tables, ring, state, n, 16, int(np.maximum(q, 0).sum()) + 300)
