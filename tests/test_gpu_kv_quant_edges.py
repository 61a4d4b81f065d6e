"""The calls on the 8-bit cache that are easy to get wrong: every way of sharing the work out, many sequences, pools past
2^32 bytes, queries that are not numbers, graphs and streams side by side, and places that do not exist."""
import ctypes

import pytest
import torch

from smolmoe_c99_b200.cache import PAGE_SIZE, LayerCache
from smolmoe_c99_b200.engine.batch import pack_step
from test_gpu_kv_quant import FORMATS, _randn, check_attention, fill, held, make_layer, ops, plain_attention, plain_rows  # noqa: F401

pytestmark = pytest.mark.gpu

HEADS = [(14, 2, 64), (28, 4, 128), (3, 1, 32), (5, 5, 48), (16, 1, 64), (16, 1, 128), (9, 1, 96), (2, 2, 16), (4, 4, 128), (2, 1, 80)]


@pytest.mark.parametrize("cluster", [0, 1, 2, 3, 4, 8])
@pytest.mark.parametrize("heads,kv_heads,hd", HEADS)
def test_every_way_to_share_a_pair_out(ops, heads, kv_heads, hd, cluster, monkeypatch):
    """The line and clusters of each size, straight from the codes whatever the step brings."""
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    monkeypatch.setattr(ops, "quant_rows_tokens", 1 << 20)
    fmt = "fp8" if (heads + cluster) % 2 else "int8"
    starts, news, slots = [0, 400, 63, 1000, 127], [1, 1, 3, 1, 20], [2, 0, 5, 1, 3]
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer(fmt, kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 60)
    for window in (0, 70):
        check_attention(ops, layer, heads, slots, starts, news, window)


@pytest.mark.parametrize("window", [0, 1, 129, 300])
@pytest.mark.parametrize("heads,kv_heads,hd", [(14, 2, 64), (28, 4, 128), (16, 1, 64), (16, 1, 128), (3, 1, 64), (4, 4, 128), (2, 2, 64), (10, 2, 128)])
def test_every_chunk_through_the_pages(ops, heads, kv_heads, hd, window, monkeypatch):
    """The tcgen05 kernel for two tokens and more: starts and ends around tiles of 64 and 128 keys, and runs that end inside
    a sequence."""
    monkeypatch.setattr(ops, "quant_rows_tokens", 1)
    fmt = "fp8" if heads % 4 else "int8"
    starts, news, slots = [0, 126, 64, 1, 640, 255], [2, 3, 64, 1, 131, 2], [4, 1, 0, 6, 2, 3]
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer(fmt, kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 61)
    check_attention(ops, layer, heads, slots, starts, news, window)


@pytest.mark.parametrize("n,cluster", [(40, None), (300, None), (700, None), (700, 0), (33, 2), (4097, None)])
def test_many_sequences(ops, n, cluster, monkeypatch):
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    ends = [1 + (37 * i) % 90 for i in range(n)]
    slots = [(n - 1 - i) for i in range(n)]
    layer = make_layer("int8", 1, 16, ends, slots)
    fill(ops, layer, slots, ends, 62)
    check_attention(ops, layer, 2, slots, [e - 1 for e in ends], [1] * n, 0)


def test_many_chunks(ops, monkeypatch):
    """More sequences that bring several tokens than one scan of a CTA takes, beside single tokens."""
    n = 450
    monkeypatch.setattr(ops, "quant_rows_tokens", 1)
    news = [1 + i % 3 for i in range(n)]
    starts = [(53 * i) % 140 for i in range(n)]
    slots = [(7 * i) % n for i in range(n)]
    ends = [s + k for s, k in zip(starts, news)]
    layer = make_layer("fp8", 1, 64, ends, slots)
    fill(ops, layer, slots, ends, 63)
    check_attention(ops, layer, 2, slots, starts, news, 0)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_pools_past_32_bits(ops, fmt):
    """Pages whose bytes lie past 2^32 in the pools, written, read back and attended to in each form."""
    pages, kv_heads, hd = (1 << 32) // (4 * PAGE_SIZE * 128) + 40, 4, 128
    starts, news, slots = [150, 0, 70], [1, 40, 3], [1, 0, 2]
    ends = [s + n for s, n in zip(starts, news)]
    pool = lambda: torch.empty((pages, kv_heads, PAGE_SIZE, hd), dtype=torch.uint8, device="cuda").view(FORMATS[fmt])
    scale = lambda: torch.full((pages, kv_heads, PAGE_SIZE), 255, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[pages - 1, 0, 0], [pages - 2, 3, pages - 9], [1, pages - 30, 0]], dtype=torch.int32, device="cuda")
    layer = LayerCache("kv", pool(), pool(), table, 0, None, k_scale=scale(), v_scale=scale())
    fill(ops, layer, [1, 2], [150, 70], 64)
    step = pack_step(slots, starts, [[0] * n for n in news], torch.device("cuda"))
    k, v = (_randn((sum(news), kv_heads, hd), s).bfloat16() for s in (65, 66))
    ops.kv_quant_store(k, v, step, layer)
    want = plain_rows(k, fmt)
    assert torch.equal(held(layer, "k", 0, 40), want[1:41]) and torch.equal(held(layer, "k", 1, 151)[150:], want[:1])
    back = ops.kv_quant_load(step, layer, torch.bfloat16)
    for i, (slot, end) in enumerate(zip(slots, ends)):
        got = back.v_pool[back.page_table[slot].long()].double().cpu().permute(0, 2, 1, 3).reshape(-1, kv_heads, hd)[:end]
        assert torch.equal(got, held(layer, "v", slot, end))
    check_attention(ops, layer, 28, slots, starts, news, 0)
    check_attention(ops, layer, 28, [1, 2], [150, 72], [1, 1], 0)


@pytest.mark.parametrize("rows_tokens", [1, 1 << 20])
def test_queries_that_are_not_numbers_touch_their_own_row_alone(ops, rows_tokens, monkeypatch):
    monkeypatch.setattr(ops, "quant_rows_tokens", rows_tokens)
    starts, news, slots = [90, 200], [7, 1], [0, 1]
    ends = [97, 201]
    layer = make_layer("fp8", 2, 64, ends, slots)
    fill(ops, layer, slots, ends, 67)
    step = pack_step(slots, starts, [[0] * n for n in news], torch.device("cuda"))
    q = _randn((8, 14, 64), 68).bfloat16()
    want, room = plain_attention(layer, q, slots, starts, news, 0.125, 0)
    q[2, 3, 5], q[7, 9, 0] = float("nan"), float("nan")
    got = ops.attention_quant(q, step, 0.125, 0, layer).double().cpu()
    ops.check_error_flag()
    spoilt = torch.zeros(8, 14, dtype=torch.bool)
    spoilt[2, 3] = spoilt[7, 9] = True
    assert torch.isnan(got[spoilt]).all()
    assert ((got - want).abs() <= room)[~spoilt].all()


@pytest.mark.parametrize("scale", [1e-6, 4.0])
@pytest.mark.parametrize("news", [[1, 1], [3, 130]])
def test_small_and_large_scales(ops, scale, news):
    starts, slots = [500, 100], [1, 0]
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer("int8", 2, 64, ends, slots)
    fill(ops, layer, slots, ends, 69)
    check_attention(ops, layer, 14, slots, starts, news, 0, scale=scale)


def test_graphs_and_streams_side_by_side(ops, monkeypatch):
    """Two captured attentions (the line; chunks through the pages) and an eager one of other sizes, at the same time on three
    streams: the same bits as one after the other."""
    def make(seed, ends, news, cluster, rows_tokens):
        slots = list(range(len(ends)))
        layer = make_layer("fp8", 4, 128, ends, slots, seed=seed)
        fill(ops, layer, slots, ends, 70 + seed)
        step = pack_step(slots, [e - n for e, n in zip(ends, news)], [[0] * n for n in news], torch.device("cuda"))
        q = _randn((sum(news), 28, 128), 80 + seed).bfloat16()

        def run():
            monkeypatch.setattr(ops, "quant_cluster", cluster)
            monkeypatch.setattr(ops, "quant_rows_tokens", rows_tokens)
            return ops.attention_quant(q, step, 0.1, 0, layer)
        return run
    runs = [make(0, [9000, 50, 4000], [1, 1, 1], 0, 8), make(1, [700, 2500], [300, 64], None, 1), make(2, [1300, 8], [2, 5], 4, 64)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for r in runs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(r())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for o in outs:
            o.fill_(float("nan"))
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = runs[2]()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])
    ops.check_error_flag()


@pytest.mark.parametrize("cluster", [0, 1, 4])
def test_pages_outside_the_pool_are_reported_by_the_attention(ops, cluster, monkeypatch):
    from smolmoe_c99_b200.kernels import KernelError
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    layer = make_layer("fp8", 2, 64, [300, 20], [0, 1])
    fill(ops, layer, [0, 1], [300, 20], 71)
    q = _randn((2, 14, 64), 72).bfloat16()
    step = pack_step([0, 1], [299, 19], [[0], [0]], torch.device("cuda"))
    want = ops.attention_quant(q, step, 0.125, 0, layer)
    for bad in (-1, layer.k_pool.shape[0]):
        kept = int(layer.page_table[0, 2])
        layer.page_table[0, 2] = bad
        got = ops.attention_quant(q, step, 0.125, 0, layer)
        with pytest.raises(KernelError, match="attention_quant met a slot, position or page outside"):
            ops.check_error_flag()
        assert torch.equal(got[1], want[1])              # (the other sequence is what it is)
        layer.page_table[0, 2] = kept
    assert torch.equal(ops.attention_quant(q, step, 0.125, 0, layer), want)
    ops.check_error_flag()


@pytest.mark.parametrize("cluster,rows_tokens", [(0, 8), (2, 8), (None, 1)])
def test_lengths_on_the_device_that_are_not_the_hosts_are_reported(ops, cluster, rows_tokens, monkeypatch):
    """A step whose sequences bring fewer tokens on the device than the host planned for: nothing is computed, the call says so,
    and the next one is what it should be."""
    from smolmoe_c99_b200.kernels import KernelError
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    monkeypatch.setattr(ops, "quant_rows_tokens", rows_tokens)
    news = [2, 60]
    layer = make_layer("fp8", 2, 64, [100, 200], [0, 1])
    fill(ops, layer, [0, 1], [100, 200], 73)
    step = pack_step([0, 1], [98, 140], [[0] * n for n in news], torch.device("cuda"))
    q = _randn((62, 14, 64), 74).bfloat16()
    want = ops.attention_quant(q, step, 0.125, 0, layer)
    cu = step.cu_seqlens.clone()
    step.cu_seqlens[1:] = torch.tensor([0, 0], dtype=torch.int32)
    ops.attention_quant(q, step, 0.125, 0, layer)
    with pytest.raises(KernelError, match="attention_quant met"):
        ops.check_error_flag()
    step.cu_seqlens.copy_(cu)
    assert torch.equal(ops.attention_quant(q, step, 0.125, 0, layer), want)
    ops.check_error_flag()


def test_a_pool_whose_memory_was_exchanged_is_read_where_it_lies_now(ops):
    layer = make_layer("int8", 2, 64, [100], [0])
    fill(ops, layer, [0], [100], 75)
    q = _randn((1, 14, 64), 76).bfloat16()
    step = pack_step([0], [99], [[0]], torch.device("cuda"))
    first = ops.attention_quant(q, step, 0.125, 0, layer)
    layer.v_pool.data = layer.v_pool.data.clone().neg_()
    assert torch.equal(ops.attention_quant(q, step, 0.125, 0, layer), -first)


def test_scales_that_are_refused(ops):
    from smolmoe_c99_b200.kernels import KernelError
    layer = make_layer("fp8", 2, 64, [100], [0])
    q, step = _randn((1, 14, 64), 77).bfloat16(), pack_step([0], [9], [[0]], torch.device("cuda"))
    for scale in (0.0, -0.125, float("nan"), float("inf")):
        with pytest.raises(KernelError, match="a scale of"):
            ops.attention_quant(q, step, scale, 0, layer)


def test_what_went_wrong_is_told_to_the_instance_that_was_called(ops):
    """Another instance of the kernel library, made later, does not receive what this one's calls have to say."""
    from smolmoe_c99_b200.kernels import KernelError, Ops
    later = Ops("plain")
    layer = make_layer("fp8", 2, 64, [200], [0])
    fill(ops, layer, [0], [200], 78)
    q, k = _randn((1, 14, 64), 79).bfloat16(), _randn((1, 2, 64), 80).bfloat16()
    step = pack_step([0], [199], [[0]], torch.device("cuda"))
    layer.page_table[0, 3] = -1
    for call, name in ((lambda: ops.kv_quant_store(k, k, step, layer), "kv_quant_store"),
                       (lambda: ops.kv_quant_load(step, layer, torch.bfloat16), "kv_quant_load"),
                       (lambda: ops.attention_quant(q, step, 0.125, 0, layer), "attention_quant")):
        call()
        later.check_error_flag()
        with pytest.raises(KernelError, match=f"{name} met"):
            ops.check_error_flag()
    ops.lib.sm_set_error_word(ctypes.c_void_p(ops._error_address))       # (as it was before `later`)
