"""The 8-bit key/value cache alone: writing it, reading it back, and the attention that reads it, against plain
computations in 64 bits. Pools start out full of bytes that stand for nothing (NaN codes, exponents without a scale),
pages lie in no order, and slots are not the numbers of the sequences."""
import math

import pytest
import torch

from smolmoe_c99_b200.cache import PAGE_SIZE, LayerCache
from smolmoe_c99_b200.engine.batch import pack_step

pytestmark = pytest.mark.gpu

FORMATS = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"fp8": 448.0, "int8": 127.0}


@pytest.fixture(scope="module")
def ops():
    from smolmoe_c99_b200.kernels import get_ops
    return get_ops()


def _randn(shape, seed, device="cuda"):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(device)


def make_layer(fmt, kv_heads, head_dim, lengths, slots, seed=0, spare=3):
    """A layer cache whose slots hold pages for ``lengths`` positions, all of it poisoned."""
    g = torch.Generator().manual_seed(seed)
    counts = [max(1, -(-n // PAGE_SIZE)) for n in lengths]
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.zeros((max(slots) + 2, max(counts)), dtype=torch.int32)
    at = 0
    for slot, n in zip(slots, counts):
        table[slot, :n] = order[at:at + n]
        at += n
    pool = lambda: torch.full((total, kv_heads, PAGE_SIZE, head_dim), 0xff, dtype=torch.uint8, device="cuda").view(FORMATS[fmt])
    scale = lambda: torch.full((total, kv_heads, PAGE_SIZE), 255, dtype=torch.uint8, device="cuda")
    return LayerCache("kv", pool(), pool(), table.cuda(), 0, None, k_scale=scale(), v_scale=scale())


def plain_rows(x, fmt):
    """What the cache stands for where it was given rows ``x``: in 64 bits, from the definition."""
    x = x.double().cpu()
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.zeros_like(amax)
    for i, a in enumerate(amax.flatten().tolist()):
        k = -100
        if math.isfinite(a) and a > 0:
            k = max(-100, math.frexp(a / TOP[fmt])[1] - 2)
            while a > TOP[fmt] * 2.0 ** k:
                k += 1
        e.view(-1)[i] = k
    step = torch.ones_like(x)
    y = x * torch.exp2(-e)
    if fmt == "fp8":
        lead = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
        lead = torch.where(torch.exp2(lead + 1) <= y.abs(), lead + 1, torch.where(torch.exp2(lead) > y.abs().clamp(min=2.0 ** -6), lead - 1, lead))
        step = torch.exp2(lead - 3)
    out = torch.round(y / step) * step * torch.exp2(e)
    return torch.where(torch.isfinite(amax), out, torch.full_like(out, float("nan")))


def held(layer, which, slot, length):
    """Positions 0..length-1 of a slot as 64-bit values [length, kv heads, head size]."""
    codes, scale = (layer.k_pool, layer.k_scale) if which == "k" else (layer.v_pool, layer.v_scale)
    pages = layer.page_table[slot, :-(-length // PAGE_SIZE)].long()
    c = codes.view(torch.uint8)[pages].view(codes.dtype).double().cpu()
    s = scale[pages].cpu()
    x = c * torch.exp2(s.double() - 127).unsqueeze(-1)
    x = torch.where((s == 255).unsqueeze(-1), torch.full_like(x, float("nan")), x)
    return x.permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:length]


def fill(ops, layer, slots, lengths, seed, k_of=None, v_of=None, dtype=torch.bfloat16):
    """Writes positions 0..length-1 of every slot; returns nothing (what is held is read from the pools)."""
    kv_heads, hd = layer.k_pool.shape[1], layer.k_pool.shape[3]
    step = pack_step(slots, [0] * len(slots), [[0] * n for n in lengths], torch.device("cuda"))
    k, v = _randn((sum(lengths), kv_heads, hd), seed), _randn((sum(lengths), kv_heads, hd), seed + 1)
    if k_of is not None:
        k = k_of(k)
    if v_of is not None:
        v = v_of(v)
    ops.kv_quant_store(k.to(dtype), v.to(dtype), step, layer)


# ---- writing and reading back -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("kv_heads,hd", [(2, 64), (4, 128), (1, 32), (5, 48), (1, 8), (3, 24), (2, 256), (1, 200)])
def test_written_and_read_back(ops, kv_heads, hd, fmt, dtype):
    slots, starts, news = [3, 0, 5], [0, 63, 130], [70, 1, 200]
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer(fmt, kv_heads, hd, ends, slots)
    fill(ops, layer, [0, 5], [63, 130], 5, dtype=dtype)
    before = {slot: (held(layer, "k", slot, n), held(layer, "v", slot, n)) for slot, n in ((0, 63), (5, 130))}
    step = pack_step(slots, starts, [[0] * n for n in news], torch.device("cuda"))
    k, v = (_randn((sum(news), kv_heads, hd), s).to(dtype) for s in (1, 2))
    k[0] = 0                                     # a row of zeros
    k[1, :, 1:] = 0                              # one value alone
    k[2] *= 2.0 ** -60
    k[3] *= 2.0 ** 90
    v[4] = v[4].abs().amax() * torch.tensor([1.0, -1.0], device="cuda").repeat(hd)[:hd]     # every code the largest
    untouched = layer.k_pool.view(torch.uint8).clone()
    rows = ops.kv_quant_store(k, v, step, layer, want_rows=True)
    pages = ops.kv_quant_load(step, layer, dtype)
    most = -(-max(ends) // PAGE_SIZE)
    assert tuple(pages.k_pool.shape) == (3 * most, kv_heads, PAGE_SIZE, hd) and pages.k_pool.dtype == dtype
    for which, x, got_rows, pool in (("k", k, rows[0], pages.k_pool), ("v", v, rows[1], pages.v_pool)):
        want = plain_rows(x, fmt)
        assert torch.equal(got_rows.double().cpu(), want), which
        first = 0
        for i, slot in enumerate(slots):
            now = held(layer, which, slot, ends[i])
            assert torch.equal(now[starts[i]:], want[first:first + news[i]]), (which, slot)
            if starts[i]:
                assert torch.equal(now[:starts[i]], before[slot][0 if which == "k" else 1])
            table = pages.page_table[slot].tolist()
            assert table == list(range(i * most, (i + 1) * most))
            back = pool[table].double().cpu().permute(0, 2, 1, 3).reshape(-1, kv_heads, hd)
            assert torch.equal(back[:ends[i]], now)
            assert not back[ends[i]:].any()      # past the end: zeros, also on pages wholly past it
            first += news[i]
    # only the pages' places of the step's positions were written
    changed = (layer.k_pool.view(torch.uint8) != untouched).flatten(2).view(untouched.shape).any(-1)
    allowed = torch.zeros_like(changed)
    for i, slot in enumerate(slots):
        for p in range(starts[i], ends[i]):
            allowed[layer.page_table[slot, p // PAGE_SIZE].long(), :, p % PAGE_SIZE] = True
    assert not (changed & ~allowed).any()
    ops.check_error_flag()


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_rounding_borders_and_ties(ops, fmt):
    """Values on and next to the borders of the grid, in float: ties go to the even code; the largest magnitude on and next
    to the border of its exponent."""
    hd = 64
    layer = make_layer(fmt, 1, hd, [256], [0])
    x = torch.zeros((256, 1, hd))
    grid = torch.tensor([m * 2.0 ** e for e in range(-9, 8) for m in (1, 1.0625, 1.125, 1.1875, 1.25, 1.3125, 1.375, 1.4375)])
    if fmt == "int8":
        grid = torch.arange(0, 127.5, 0.5)
    up, down = torch.nextafter(grid, torch.tensor(1e9)), torch.nextafter(grid, torch.tensor(-1e9))
    for i in range(250):
        x[i, 0, 0] = TOP[fmt]
        picked = torch.arange(hd - 1) + i * 7
        x[i, 0, 1:] = torch.stack([grid, up, down], 1).flatten()[picked % (3 * len(grid))] * (-1.0) ** i
        x[i] *= 2.0 ** (i % 40 - 20)
    for j, top in enumerate([TOP[fmt], TOP[fmt] / 2]):
        for k, move in enumerate([0.0, 1e9, -1e9]):
            x[250 + 3 * j + k, 0, 0] = torch.nextafter(torch.tensor(top), torch.tensor(move)) if move else top
            x[250 + 3 * j + k, 0, 1] = 1.0
    step = pack_step([0], [0], [[0] * 256], torch.device("cuda"))
    rows = ops.kv_quant_store(x.cuda(), -x.cuda(), step, layer, want_rows=True)
    want = plain_rows(x, fmt)
    assert torch.equal(rows[0].double().cpu(), want)
    assert torch.equal(rows[1].double().cpu(), -want)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_rows_without_a_scale(ops, fmt):
    """A row with an infinity or a NaN reads back as NaN whole; its neighbours are what they are."""
    layer = make_layer(fmt, 2, 64, [10], [1])
    k = _randn((10, 2, 64), 3).bfloat16()
    k[2, 0, 5], k[4, 1, 63], k[6, 0, 0] = float("inf"), float("nan"), float("-inf")
    step = pack_step([1], [0], [[0] * 10], torch.device("cuda"))
    rows = ops.kv_quant_store(k, k.flip(0), step, layer, want_rows=True)
    want = plain_rows(k, fmt)
    assert torch.equal(torch.nan_to_num(rows[0].double().cpu(), nan=1e30), torch.nan_to_num(want, nan=1e30))
    assert int(torch.isnan(rows[0]).all(-1).sum()) == 3
    pages = ops.kv_quant_load(step, layer, torch.float32)
    back = pages.v_pool[0].permute(1, 0, 2)[:10].flip(0).double().cpu()
    assert torch.equal(torch.nan_to_num(back, nan=1e30), torch.nan_to_num(want, nan=1e30))


def test_places_outside_the_cache_are_left_out_and_reported(ops):
    from smolmoe_c99_b200.kernels import KernelError
    layer = make_layer("fp8", 2, 64, [64], [0])
    k = _randn((1, 2, 64), 3).bfloat16()
    for spoil in ("page", "position", "slot"):
        step = pack_step([0], [3], [[0]], torch.device("cuda"))
        table = layer.page_table.clone()
        if spoil == "page":
            layer.page_table[0, 0] = layer.k_pool.shape[0]
        elif spoil == "position":
            step.positions[0] = 64 * layer.page_table.shape[1]
        else:
            step.token_slot[0] = layer.page_table.shape[0]
        before = layer.k_pool.view(torch.uint8).clone()
        ops.kv_quant_store(k, k, step, layer)
        assert torch.equal(layer.k_pool.view(torch.uint8), before)
        with pytest.raises(KernelError, match="kv_quant_store met a slot, position or page outside"):
            ops.check_error_flag()
        layer.page_table.copy_(table)
    layer.page_table[0, 0] = -1
    ops.kv_quant_load(pack_step([0], [3], [[0]], torch.device("cuda")), layer, torch.bfloat16)
    with pytest.raises(KernelError, match="kv_quant_load met"):
        ops.check_error_flag()
    ops.check_error_flag()


# ---- attention ----------------------------------------------------------------------------------------------------------

def plain_attention(layer, q, slots, starts, news, scale, window):
    """In 64 bits: the output, and how far a kernel may be off: half a step of the output's type, a relative half step of
    bfloat16 for each weight (which kernels hold in 16 bits), and what sums of head-size products in float move a score.
    A weight so far below the largest that its form has no number for it may be lost: float has none below 2^-126 of the
    largest (a softmax's largest weight is 1); a half-precision weight that carries its row's scale, put at 2^15 for the
    largest weight and scale, has steps of 2^-24, so half a step is 2^-40 of the largest value a key of that scale adds. Each
    of the n keys can lose that much (times the largest magnitude of a value, whose code is at most twice its scale's
    largest: 2^-39)."""
    heads, hd = q.shape[1], q.shape[2]
    kv_heads = layer.k_pool.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64)
    room = torch.empty(q.shape, dtype=torch.float64)
    half = torch.finfo(q.dtype).eps / 2
    least = 2.0 ** -39 if q.dtype == torch.bfloat16 else 2.0 ** -125
    weight = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    qd = q.double().cpu()
    first = 0
    for slot, s, n in zip(slots, starts, news):
        k, v = held(layer, "k", slot, s + n), held(layer, "v", slot, s + n)
        for h in range(heads):
            kh, vh, x = k[:, h // (heads // kv_heads)], v[:, h // (heads // kv_heads)], qd[first:first + n, h]
            scores = x @ kh.T * scale
            moved = (hd + 8) * 2.0 ** -24 * float((x.abs() @ torch.nan_to_num(kh).abs().T * scale).max())
            pos, key = torch.arange(s, s + n).view(-1, 1), torch.arange(s + n)
            seen = (key <= pos) & ((key > pos - window) if window else torch.ones(()).bool())
            for i in range(n):      # (row by row: what a row does not see must not touch it, NaN or not)
                p = torch.softmax(scores[i][seen[i]], 0)
                out[first + i, h] = p @ vh[seen[i]]
                spread = p @ vh[seen[i]].abs()
                lost = least * int(seen[i].sum()) * float(torch.nan_to_num(vh).abs().max())
                room[first + i, h] = half * out[first + i, h].abs() + (weight + 2 * moved + 2.0 ** -18) * spread + lost
        first += n
    return out, room


def check_attention(ops, layer, heads, slots, starts, news, window, dtype=torch.bfloat16, seed=9, scale=None, q=None):
    hd = layer.k_pool.shape[3]
    scale = hd ** -0.5 if scale is None else scale
    step = pack_step(slots, starts, [[0] * n for n in news], torch.device("cuda"))
    if q is None:
        q = (_randn((sum(news), heads, hd), seed) * 1.5).to(dtype)
    got = ops.attention_quant(q, step, scale, window, layer)
    ops.check_error_flag()
    want, room = plain_attention(layer, q, slots, starts, news, scale, window)
    assert got.dtype == q.dtype and got.shape == q.shape
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    off = torch.where(got == want, torch.zeros_like(room), (got - want).abs() / room)[fine]   # (a sum of zeros has no room)
    assert off.numel() == 0 or float(off.max()) <= 1.0, f"{float(off.max()):.3g} of what rounding can move"
    return got


HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (6, 3, 64), (3, 1, 32), (5, 5, 48), (16, 1, 64), (8, 1, 128), (9, 1, 96), (2, 2, 16)]


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads,kv_heads,hd", HEADS)
def test_single_tokens(ops, heads, kv_heads, hd, fmt):
    """Decode: lengths around the pages' and tiles' edges, and of one position."""
    ends = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 300, 511, 700]
    slots = [(7 * i) % len(ends) for i in range(len(ends))]
    layer = make_layer(fmt, kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 20)
    check_attention(ops, layer, heads, slots, [e - 1 for e in ends], [1] * len(ends), 0)
    check_attention(ops, layer, heads, slots[:1], [ends[0] - 1], [1], 0)
    check_attention(ops, layer, heads, slots[-1:], [ends[-1] - 1], [1], 0)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
@pytest.mark.parametrize("heads,kv_heads,hd", [(14, 2, 64), (8, 2, 128), (3, 1, 32)])
def test_single_tokens_in_a_window(ops, heads, kv_heads, hd, window, fmt):
    ends = [1, 5, 6, 64, 65, 99, 100, 101, 164, 165, 400, 999]
    slots = list(reversed(range(len(ends))))
    layer = make_layer(fmt, kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 21)
    check_attention(ops, layer, heads, slots, [e - 1 for e in ends], [1] * len(ends), window)


@pytest.mark.parametrize("heads,kv_heads,hd,ends", [(14, 2, 64, [5000, 3, 1200]), (28, 4, 128, [9000]), (6, 3, 64, [12345, 77]),
                                                    (4, 4, 80, [3001, 2999])])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_single_tokens_of_long_sequences(ops, heads, kv_heads, hd, ends, fmt):
    slots = list(range(1, len(ends) + 1))
    layer = make_layer(fmt, kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 22)
    check_attention(ops, layer, heads, slots, [e - 1 for e in ends], [1] * len(ends), 0)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("window", [0, 1, 50, 200])
@pytest.mark.parametrize("heads,kv_heads,hd", [(14, 2, 64), (12, 2, 128), (6, 3, 64), (3, 1, 32), (5, 5, 48), (9, 1, 96), (2, 2, 16)])
def test_chunks(ops, heads, kv_heads, hd, window, fmt):
    """Sequences at their start, one token each, a few and many, in one step."""
    starts, news = [0, 100, 63, 200, 1, 128, 0, 300], [5, 1, 2, 9, 64, 65, 1, 130]
    slots = [5, 2, 7, 0, 1, 9, 3, 4]
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer(fmt, kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 23)
    check_attention(ops, layer, heads, slots, starts, news, window)


@pytest.mark.parametrize("heads,kv_heads,hd,start,new", [(14, 2, 64, 1000, 3), (14, 2, 64, 2000, 17), (14, 2, 64, 700, 300), (28, 4, 128, 1100, 40),
                                                         (12, 2, 128, 0, 500), (6, 3, 64, 777, 200), (4, 2, 128, 3000, 129), (14, 2, 64, 0, 1)])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_one_chunk(ops, heads, kv_heads, hd, start, new, fmt):
    layer = make_layer(fmt, kv_heads, hd, [start + new], [1])
    fill(ops, layer, [1], [start + new], 24)
    check_attention(ops, layer, heads, [1], [start], [new], 0)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_attention_in_float(ops, fmt):
    """The 32-bit path, and head sizes that no tensor-core kernel takes."""
    for heads, kv_heads, hd in [(4, 2, 64), (3, 1, 24), (2, 1, 256)]:
        starts, news, slots = [0, 80, 129], [70, 1, 3], [2, 0, 1]
        ends = [s + n for s, n in zip(starts, news)]
        layer = make_layer(fmt, kv_heads, hd, ends, slots)
        fill(ops, layer, slots, ends, 25, dtype=torch.float32)
        check_attention(ops, layer, heads, slots, starts, news, 0, torch.float32)
        check_attention(ops, layer, heads, slots, starts, news, 33, torch.float32)
        check_attention(ops, layer, heads, slots, starts, news, 0, torch.bfloat16)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("news", [[1, 1, 1], [20, 1, 7], [200, 1, 150]])
def test_rows_of_very_unequal_size(ops, news, fmt):
    """Keys and values whose rows differ by many powers of two (each has a scale of its own), a key that dominates late,
    and query rows of tiny and of huge values."""
    starts, slots = [300, 1000, 400], [0, 1, 2]
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer(fmt, 2, 64, ends, slots)
    sizes = torch.exp2(torch.randint(-12, 3, (sum(ends), 2, 1), generator=torch.Generator().manual_seed(4)).float()).cuda()

    def keys(k):
        k = k * sizes
        k[-40] = k[-40].sign() * 6.0
        return k
    fill(ops, layer, slots, ends, 26, keys, lambda v: v * sizes.flip(0))
    q = _randn((sum(news), 14, 64), 27) * 2
    q[0] *= 2.0 ** -30
    q[-1] *= 2.0 ** 4
    check_attention(ops, layer, 14, slots, starts, news, 0, q=q.bfloat16())


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("news", [[1, 1], [6, 30], [180, 200]])
def test_what_a_row_does_not_see_does_not_touch_it(ops, news, fmt):
    """Rows of keys and values that read back as NaN, before a window and behind a token's position: the tokens that see
    them are NaN, the others are what they would be without."""
    starts, slots, window = [300, 129], [1, 0], 90
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer(fmt, 2, 64, ends, slots)

    def spoil(x):
        for base, s, n in ((0, starts[0], news[0]), (ends[0], starts[1], news[1])):
            for p in (0, 20, s - 100, s - window):           # no token of the step sees these
                x[base + p, 0, 3] = float("nan")
            x[base + s + n - 1, 1, 7] = float("inf")        # the last token alone sees this one
        return x
    fill(ops, layer, slots, ends, 28, spoil, spoil)
    got = check_attention(ops, layer, 14, slots, starts, news, window)
    nan = torch.isnan(got).any(-1)
    assert not nan[:, :7].any()
    last = torch.tensor([news[0] - 1, sum(news) - 1])
    assert nan[last, 7:].all() and int(nan.sum()) == 14


def test_the_same_inputs_give_the_same_bits(ops):
    ends, slots = [3000, 100, 777, 1500], [0, 1, 2, 3]
    layer = make_layer("fp8", 2, 64, ends, slots)
    fill(ops, layer, slots, ends, 29)
    for news in ([1, 1, 1, 1], [3, 1, 10, 200]):
        step = pack_step(slots, [e - n for e, n in zip(ends, news)], [[0] * n for n in news], torch.device("cuda"))
        q = _randn((sum(news), 14, 64), 30).bfloat16()
        outs = [ops.attention_quant(q, step, 0.125, 0, layer) for _ in range(5)]
        assert all(torch.equal(o, outs[0]) for o in outs)


def test_written_read_and_attended_in_a_graph_and_on_another_stream(ops):
    """A run of them as a layer makes them, captured and replayed with other numbers, beside an eager run of another size
    on another stream."""
    ends, slots = [200, 513], [1, 0]
    layer, other = (make_layer("fp8", 2, 64, ends, slots, seed=s) for s in (0, 1))
    news = [1, 1]
    starts = [e - 1 for e in ends]

    def run(k, v, q, step, where):
        ops.kv_quant_store(k, v, step, where)
        return ops.attention_quant(q, step, 0.125, 0, where)
    for where in (layer, other):
        fill(ops, where, slots, ends, 31)
    step = pack_step(slots, starts, [[0]] * 2, torch.device("cuda"))
    k, v, q = (_randn((2, h, 64), 40 + h).bfloat16() for h in (2, 2, 14))
    run(k, v, q, step, layer)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(k, v, q, step, layer)
    side = torch.cuda.Stream()
    for seed in (1, 2, 3):
        k.copy_(_randn((2, 2, 64), 50 + seed))
        q.copy_(_randn((2, 14, 64), 60 + seed))
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            more = run(k, v, q, step, other)
        torch.cuda.current_stream().wait_stream(side)
        want, room = plain_attention(layer, q, slots, starts, news, 0.125, 0)
        assert ((out.double().cpu() - want).abs() <= room).all()
        want, room = plain_attention(other, q, slots, starts, news, 0.125, 0)
        assert ((more.double().cpu() - want).abs() <= room).all()


def test_refusals(ops):
    from smolmoe_c99_b200.kernels import KernelError
    layer = make_layer("fp8", 2, 64, [100], [0])
    step = pack_step([0], [9], [[0]], torch.device("cuda"))
    q, k = _randn((1, 14, 64), 1).bfloat16(), _randn((1, 2, 64), 2).bfloat16()
    with pytest.raises(KernelError, match="expected 1 tokens"):
        ops.attention_quant(q.repeat(2, 1, 1), step, 0.125, 0, layer)
    with pytest.raises(KernelError, match="multiple of 2 heads"):
        ops.attention_quant(q[:, :13].contiguous(), step, 0.125, 0, layer)
    with pytest.raises(KernelError, match="contiguous"):
        ops.attention_quant(q.repeat(1, 2, 1)[:, ::2], step, 0.125, 0, layer)
    with pytest.raises(KernelError, match="unsupported dtype|float32 or bfloat16"):
        ops.attention_quant(q.half(), step, 0.125, 0, layer)
    with pytest.raises(KernelError, match="window"):
        ops.attention_quant(q, step, 0.125, -3, layer)
    with pytest.raises(KernelError, match="packed"):
        ops.kv_quant_store(k, k[:, :1].contiguous(), step, layer)
    with pytest.raises(KernelError, match="packed values"):
        ops.kv_quant_store(k, k.float(), step, layer)
    with pytest.raises(KernelError, match="unsupported dtype"):
        ops.kv_quant_store(k.half(), k.half(), step, layer)
    with pytest.raises(KernelError, match="read back as"):
        ops.kv_quant_load(step, layer, torch.float16)
    with pytest.raises(KernelError, match="8-bit"):
        ops.kv_quant_load(step, LayerCache("kv", k, k, layer.page_table), torch.bfloat16)
