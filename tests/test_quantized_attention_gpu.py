"""quantized_ragged_page_attention on the GPU against the float64 evaluation."""

import numpy as np
import pytest
import torch

from ejkernel_amd.modules import quantized_ragged_page_attention
from tests.quantized_helpers import Batch

pytestmark = pytest.mark.gpu

KINDS = ("int8", "e4m3", "e5m2")


def run(b):
    out = quantized_ragged_page_attention(*b.args(), **b.kwargs())
    torch.cuda.synchronize()
    b.check(out)
    return out


SHAPES = {  # q_heads, kv_heads, dim, page, block
    "d128": (8, 2, 128, 16, 16), "d64": (6, 2, 64, 32, 8), "d256": (4, 2, 256, 16, 4), "d96": (4, 1, 96, 64, 32),
    "d80": (5, 5, 80, 4, 4), "d16": (3, 1, 16, 8, 4), "d192": (8, 1, 192, 128, 64), "d240": (2, 2, 240, 8, 8), "d48": (14, 2, 48, 256, 128),
}


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_decode_and_chunks(shape, kind, dtype):
    q_heads, kv_heads, dim, page, block = SHAPES[shape]
    seqs = [(1, 1), (1, 33), (2, 2), (1, 700), (0, 40), (3, 129), (37, 37), (1, 31), (70, 300), (1, 0), (5, 64), (1, 257)]
    run(Batch(seqs, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, block=block, kind=kind, dtype=dtype, slack=5, spare_seqs=2,
              seed=dim + page))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("window,cap,sinks", [(1, None, 0), (7, None, 2), (100, 20.0, 0), (None, 5.0, 1), (333, None, 3), (None, None, 1), (64, 30.0, 5)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_window_cap_and_sinks(dim, window, cap, sinks, dtype):
    seqs = [(1, 900), (4, 500), (1, 5), (150, 400), (1, 0), (33, 33), (2, 64), (0, 7), (20, 1000)]
    run(Batch(seqs, q_heads=8, kv_heads=2, dim=dim, page=16, block=8, kind="int8" if window else "e4m3", dtype=dtype, window=window,
              cap=cap, sinks=sinks, slack=2, seed=dim + sinks))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs", [[(1, 5000)], [(1, 20001), (1, 3)], [(1, 1)], [(2, 9000), (1, 8191), (1, 8192), (1, 8193)],
                                  [(300, 2300)], [(513, 513)], [(129, 4000), (1, 4000)], [(1, n) for n in range(0, 140)]],
                         ids=["one_long", "long_and_short", "one_key", "few_long", "one_chunk", "from_scratch", "chunk_beside", "every_length"])
def test_splits(seqs, kind):
    run(Batch(seqs, q_heads=8, kv_heads=2, dim=128, page=16, block=16, kind=kind, seed=len(seqs)))


@pytest.mark.parametrize("group", [1, 2, 3, 7, 16, 17, 40, 65, 130, 200])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_group_sizes(group, dtype):
    run(Batch([(1, 200), (3, 77), (6, 6), (40, 90), (1, 1)], q_heads=2 * group, kv_heads=2, dim=64, page=16, block=4, kind="e4m3", dtype=dtype, seed=group))


@pytest.mark.parametrize("page,block", [(4, 4), (8, 4), (8, 8), (32, 4), (64, 64), (512, 4), (512, 512), (2048, 16)])
def test_pages_and_blocks(page, block):
    run(Batch([(1, 300), (60, 130), (1, 4), (2, 1025)], q_heads=4, kv_heads=1, dim=128, page=page, block=block, kind="int8", seed=page + block))


def test_many_sequences():
    rng = np.random.default_rng(3)
    seqs = [(int(q), int(q + k)) for q, k in zip(rng.choice([0, 1, 1, 1, 2, 9], size=2500), rng.integers(0, 60, size=2500))]
    run(Batch(seqs, q_heads=2, kv_heads=1, dim=64, page=8, block=8, kind="e5m2", slack=9, seed=4))


def test_negative_and_zero_scale():
    for scale in (-0.2, 0.0, 3.0):
        run(Batch([(1, 100), (40, 50)], q_heads=4, kv_heads=2, dim=64, page=16, block=16, kind="int8", scale=scale, seed=1))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_negative_scale_of_large_logits(dtype):
    """Logits of thousands of either sign: the running maximum has to follow the scaled ones, not the products."""
    run(Batch([(1, 300), (3, 90), (70, 150)], q_heads=4, kv_heads=2, dim=64, page=16, block=16, kind="int8", dtype=dtype, scale=-40.0, seed=3))
    run(Batch([(1, 300), (70, 150)], q_heads=4, kv_heads=2, dim=64, page=8, block=8, kind="e4m3", dtype=dtype, scale=-40.0, cap=900.0, seed=4))


def test_largest_window_is_no_window():
    """Requests that have more tokens than keys, too: their first rows lie in front of every key."""
    b = Batch([(1, 70), (60, 100), (33, 33)], q_heads=4, kv_heads=2, dim=64, page=16, block=16, kind="int8", seed=6)
    want = run(b)
    assert torch.equal(quantized_ragged_page_attention(*b.args(), softmax_scale=b.scale, sliding_window=2**31 - 1), want)
    lens = b.args()[3] // 2  # the pages stay whose keys these are
    args = [*b.args()[:3], lens, *b.args()[4:]]
    want = quantized_ragged_page_attention(*args)
    assert torch.isfinite(want).all()
    assert torch.equal(quantized_ragged_page_attention(*args, sliding_window=2**31 - 1), want)


def test_extreme_logits_and_scales():
    """Logits of thousands, scales next to the least and the largest that an update makes, blocks of zeros."""
    b = Batch([(1, 200), (50, 120)], q_heads=4, kv_heads=2, dim=64, page=16, block=16, kind="e4m3", dtype="fp32", seed=2, scale=20.0)
    b.scales[:, 1::2] = np.where(np.isnan(b.scales[:, 1::2]), np.nan, 2.0**-126)
    b.scales[::3, 1::2] = np.where(np.isnan(b.scales[::3, 1::2]), np.nan, 2.0**74)
    b.scales[:, 0::2][::4] *= 0
    run(b)


def test_queries_are_read_in_place_from_a_fused_projection():
    b = Batch([(1, 90), (3, 50), (40, 41), (1, 7)], q_heads=4, kv_heads=2, dim=128, page=16, block=16, kind="int8", seed=5)
    want = run(b)
    args = list(b.args())
    t = args[0].shape[0]
    fused = torch.randn((t, 8, 128), device="cuda:0").to(torch.bfloat16)
    fused[:, :4] = args[0]
    args[0] = fused[:, :4]
    assert torch.equal(quantized_ragged_page_attention(*args, **b.kwargs()), want)
    flipped = b.args()[0].transpose(0, 1).contiguous().transpose(0, 1)  # head-major memory
    args[0] = flipped
    assert torch.equal(quantized_ragged_page_attention(*args, **b.kwargs()), want)
    odd = torch.empty(t * 4 * 128 + 1, dtype=torch.bfloat16, device="cuda:0")[1:].view(t, 4, 128)  # rows off the 16-byte grid
    odd.copy_(b.args()[0])
    args[0] = odd
    assert torch.equal(quantized_ragged_page_attention(*args, **b.kwargs()), want)


def test_repeated_calls_and_streams_agree_bit_for_bit():
    b = Batch([(1, 3000), (1, 100), (200, 700), (1, 0), (4, 4000)], q_heads=8, kv_heads=2, dim=128, page=16, block=16, kind="e4m3", seed=6)
    args = b.args()
    want = quantized_ragged_page_attention(*args, **b.kwargs())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for k in range(9):
        with torch.cuda.stream(streams[k % 3]):
            outs.append(quantized_ragged_page_attention(*args, **b.kwargs()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    b.check(want)


def test_two_graphs_replayed_beside_eager_calls():
    """Two captured calls of other shapes, replayed in turn with eager calls between and their inputs changed in place."""
    batches = [Batch([(1, 3000), (5, 100), (1, 1)], q_heads=8, kv_heads=2, dim=128, page=16, block=16, kind="int8", seed=7),
               Batch([(1, 50), (300, 700)], q_heads=8, kv_heads=2, dim=128, page=16, block=16, kind="int8", seed=8)]
    args = [b.args() for b in batches]
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        for a, b in zip(args, batches):
            quantized_ragged_page_attention(*a, **b.kwargs())
        torch.cuda.synchronize()
        for a, b in zip(args, batches):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                outs.append(quantized_ragged_page_attention(*a, **b.kwargs()))
            graphs.append(g)
    torch.cuda.synchronize()
    for k in range(4):
        for a, b in zip(args, batches):
            b.queries = b.queries.roll(1, 0) if k else b.queries
            a[0].copy_(b.queries)
        for g in graphs:
            g.replay()
        eager = [quantized_ragged_page_attention(*a, **b.kwargs()) for a, b in zip(args, batches)]
        torch.cuda.synchronize()
        for o, e, b in zip(outs, eager, batches):
            assert torch.equal(o, e)
            b.check(o)


def test_malformed_device_metadata_stays_in_bounds():
    """Lengths, starts, counts and pages that no batch has: the call ends and writes nothing but its output."""
    b = Batch([(1, 60), (40, 90), (2, 30)], q_heads=4, kv_heads=2, dim=64, page=16, block=16, kind="int8", seed=9)
    for lens, starts, count in (([1 << 30, -5, 70], [0, 1, 41, 43], 3), ([60, 90, 30], [0, 50, 7, 1 << 30], 3), ([60, 90, 30], [-4, 1, 41, 43], 99),
                                ([60, 90, 30], [0, 1, 41, 43], -1), ([60, 90, 10], [0, 1, 41, 43], 3)):
        args = list(b.args())
        args[3] = torch.tensor(lens, dtype=torch.int32, device="cuda:0")
        args[5] = torch.tensor(starts, dtype=torch.int32, device="cuda:0")
        args[6] = torch.tensor([count], dtype=torch.int32, device="cuda:0")
        before = [a.clone() for a in args[1:]]
        out = quantized_ragged_page_attention(*args, **b.kwargs())
        torch.cuda.synchronize()
        assert out.shape == args[0].shape
        assert all(torch.equal(x.view(torch.uint8) if x.dtype.itemsize == 1 else x.nan_to_num(), y.view(torch.uint8) if y.dtype.itemsize == 1 else y.nan_to_num())
                   for x, y in zip(before, args[1:]))
    b.check(quantized_ragged_page_attention(*b.args(), **b.kwargs()))


@pytest.mark.parametrize("seqs,heads", [(60, 8), (64, 8), (65, 8), (32, 8), (33, 8), (29, 16), (256, 2), (512, 1), (3, 2)])
def test_items_as_many_as_workgroups(seqs, heads):
    """Around half and the whole of the workgroups that 256 compute units take: whole items, equal parts, cuts anywhere."""
    for lens in ([500] * seqs, [40 + 13 * k % 700 for k in range(seqs)], [3000] + [30] * (seqs - 1)):
        run(Batch([(1, n) for n in lens], q_heads=heads, kv_heads=heads, dim=16, page=64, block=16, kind="int8", seed=seqs))


def test_two_threads_on_streams_of_their_own():
    import threading

    batches = [Batch([(1, 3000), (50, 700), (1, 5)], q_heads=8, kv_heads=2, dim=64, page=16, block=16, kind="int8", seed=1),
               Batch([(1, 900)] * 20 + [(200, 200)], q_heads=8, kv_heads=2, dim=128, page=16, block=16, kind="e4m3", seed=2)]
    args = [b.args() for b in batches]
    want = [run(b) for b in batches]
    same, errors = [[], []], []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(25):
                    same[k].append(torch.equal(quantized_ragged_page_attention(*args[k], **batches[k].kwargs()), want[k]))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and all(len(s) == 25 and all(s) for s in same), errors


def test_soft_cap_in_fp32_keeps_fp32_logits():
    """Two keys, the first of logit 0, whose log-odds give the second's capped logit back.

    It takes nine roundings of its own size (the products' sum, scales, 1 / cap and its product, tanh, cap), each off by 2**-24 / sqrt(3) in
    the mean square: 4.5 * 3 * 2**-24 / sqrt(3) = 4.7e-7 at most.  The exponential's argument adds 1.5e-7, its value and the
    output's division and rounding 1e-7: 5.1e-7 in all.  A tanh that is off by 6e-8 of the cap would add 1.3e-6.
    """
    rng = np.random.default_rng(0)
    seqs, heads, dim, cap = 1024, 4, 16, 30.0
    codes = np.zeros((1, 2 * heads, 16, dim), np.int8)
    codes[0, 0::2, 1, 3] = 1
    codes[0, 1::2, 1, :] = 1
    x = torch.zeros((seqs, heads, dim))
    x[:, :, 3] = torch.from_numpy(-cap * rng.uniform(0.0625, 0.15, size=(seqs, heads))).float()
    out = quantized_ragged_page_attention(x.to("cuda:0"), torch.from_numpy(codes).to("cuda:0"), torch.ones((1, 2 * heads, 1), device="cuda:0"),
                                          torch.full((seqs,), 2, dtype=torch.int32, device="cuda:0"), torch.zeros((seqs, 1), dtype=torch.int32, device="cuda:0"),
                                          torch.arange(seqs + 1, dtype=torch.int32, device="cuda:0"), seqs, softmax_scale=1.0, logits_soft_cap=cap)
    p = out[:, :, 5].double().cpu().numpy()
    off = np.log(p / (1 - p)) - cap * np.tanh(x[:, :, 3].double().numpy() / cap)
    assert np.sqrt((off**2).mean()) < 7.5e-7
