"""Calls on the 8-bit cache at the ends of what they take: values of very unequal size, long chunks, many sequences, lengths and
windows at the borders of their types."""
import pytest
import torch

from smolmoe_c99_b200.engine.batch import pack_step
from test_gpu_kv_quant import _randn, fill, held, make_layer, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def row_by_row(layer, q, slots, starts, news, scale, window):
    """The output in 64 bits and how far a kernel may be off, each row from what it sees alone. Half a step of the output (2^-8
    for bfloat16); half a step of a bfloat16 weight (2^-8; half precision has 2^-11); what float sums of head-size products move
    a score by, twice (numerator and denominator); 2^-18 for float sums of up to 2^5 parts of the weighted values. A half-precision
    weight is P 2^e put between 2^8 and 2^15 for the row's largest (e the exponent of the value row's scale) and ends in steps
    of 2^-24, so each of the n weights may be off by 2^-25 / 2^8 = 2^-33 of the largest P 2^e, and a value is a code of at most
    448 (127) times 2^e, at most twice the largest magnitude of a row of that scale: 2^-32 of the largest P amax."""
    heads, kv_heads = q.shape[1], layer.k_pool.shape[1]
    hd = q.shape[2]
    out, room = torch.empty(q.shape, dtype=torch.float64), torch.empty(q.shape, dtype=torch.float64)
    qd, first = q.double().cpu(), 0
    for slot, s, n in zip(slots, starts, news):
        k, v = held(layer, "k", slot, s + n), held(layer, "v", slot, s + n)
        for i in range(n):
            lo = max(0, s + i - window + 1) if window else 0
            for h in range(heads):
                kh, vh, x = (t[lo:s + i + 1, h // (heads // kv_heads)] for t in (k, v, k))
                x = qd[first + i, h]
                p = torch.softmax(kh @ x * scale, 0)
                moved = (hd + 8) * 2.0 ** -24 * float((kh.abs() @ x.abs()).max()) * scale
                spread = p @ vh.abs()
                lost = 2.0 ** -32 * len(p) * float((p * vh.abs().amax(-1)).max())
                out[first + i, h] = p @ vh
                room[first + i, h] = 2.0 ** -8 * out[first + i, h].abs() + (2.0 ** -8 + 2 * moved + 2.0 ** -18) * spread + lost
        first += n
    return out, room


def check_rows(ops, layer, q, slots, starts, news, scale, window):
    step = pack_step(slots, starts, [[0] * n for n in news], torch.device("cuda"))
    got = ops.attention_quant(q, step, scale, window, layer).double().cpu()
    ops.check_error_flag()
    want, room = row_by_row(layer, q, slots, starts, news, scale, window)
    off = (got - want).abs() / room
    assert float(off.max()) <= 1.0, f"{float(off.max()):.3g} of what rounding can move"


# ---- value rows of very unequal size ------------------------------------------------------------------------------------

@pytest.mark.parametrize("power", [30, 45, 90])
@pytest.mark.parametrize("cluster,rows_tokens", [(None, 64), (0, 64), (4, 64), (None, 1)])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(14, 2, 64), (8, 1, 128)])
def test_large_values_that_a_row_does_not_see(ops, heads, kv_heads, hd, fmt, cluster, rows_tokens, power, monkeypatch):
    """The last token of each chunk, and the position that leaves the window with the second, have values 2^power times the
    others'."""
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    monkeypatch.setattr(ops, "quant_rows_tokens", rows_tokens)
    starts, news, slots, window = [70, 200], [4, 9], [1, 0], 50
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer(fmt, kv_heads, hd, ends, slots)

    def enlarge(v):
        for base, s, n in ((0, starts[0], news[0]), (ends[0], starts[1], news[1])):
            v[base + s + n - 1] *= 2.0 ** power
            v[base + s - window + 1] *= 2.0 ** power
        return v
    fill(ops, layer, slots, ends, 90, v_of=enlarge)
    q = _randn((sum(news), heads, hd), 91).bfloat16()
    check_rows(ops, layer, q, slots, starts, news, hd ** -0.5, window)
    check_rows(ops, layer, q, slots, starts, news, hd ** -0.5, 0)


@pytest.mark.parametrize("power", [30, 45, 90])
@pytest.mark.parametrize("cluster", [None, 0, 4])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_large_values_without_weight(ops, fmt, cluster, power, monkeypatch):
    """Positions whose values are 2^power times the others' and whose scores lie 2^-140 and less below the largest, met before,
    among and after the others; then scores that rise from position to position, with values that fall."""
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    n, hd = 500, 64
    layer = make_layer(fmt, 2, hd, [n], [0])
    q = (_randn((1, 2, hd), 92).abs() + 0.5).bfloat16()

    def keys(k):
        k *= 0.25
        for p in (0, 40, 255, 499):
            k[p] = -8.0
        return k

    def values(v):
        for p in (0, 40, 255, 499):
            v[p] *= 2.0 ** power
        return v
    fill(ops, layer, [0], [n], 93, keys, values)
    check_rows(ops, layer, q, [0], [n - 1], [1], 0.25, 0)
    rise = torch.linspace(-10, 10, n, device="cuda").view(-1, 1, 1)
    fall = torch.exp2(torch.linspace(power, -power, n, device="cuda")).view(-1, 1, 1)
    fill(ops, layer, [0], [n], 94, lambda k: k * 0.1 + rise, lambda v: v * fall)
    check_rows(ops, layer, q, [0], [n - 1], [1], 0.25, 0)


@pytest.mark.parametrize("cluster,rows_tokens", [(None, 64), (0, 64), (4, 64), (1, 64)])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("rising", [True, False])
def test_values_over_all_that_a_scale_can_be(ops, fmt, rising, cluster, rows_tokens, monkeypatch):
    """Equal scores, values from 2^-88 to 2^118 in runs of 40 positions: sums of weights count every position alike, however little its
    values add. Then the least values alone, and the largest alone."""
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    monkeypatch.setattr(ops, "quant_rows_tokens", rows_tokens)
    n, hd = 1000, 64
    layer = make_layer(fmt, 2, hd, [n], [0])
    q = _randn((2, 4, hd), 112).bfloat16()
    power = torch.linspace(-88, 118, 25).round().repeat_interleave(40)[:n]
    for powers in (power if rising else power.flip(0), torch.full((n,), -98.0), torch.full((n,), 118.0)):
        fill(ops, layer, [0], [n], 113, lambda k: k * 0.02, lambda v: v.clamp(-4, 4) * torch.exp2(powers).view(-1, 1, 1).cuda())
        check_rows(ops, layer, q, [0], [n - 2], [2], 0.125, 0)


# ---- windows ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows_tokens", [64, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_windows_wider_than_any_sequence_see_all(ops, dtype, rows_tokens, monkeypatch):
    monkeypatch.setattr(ops, "quant_rows_tokens", rows_tokens)
    starts, news, slots = [300, 128, 0], [1, 40, 3], [2, 0, 1]
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer("fp8", 2, 64, ends, slots)
    fill(ops, layer, slots, ends, 95)
    q = _randn((sum(news), 4, 64), 96).to(dtype)
    step = pack_step(slots, starts, [[0] * n for n in news], torch.device("cuda"))
    want = ops.attention_quant(q, step, 0.125, 0, layer)
    for window in (10_000, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 32 + 5, 2 ** 40):
        assert torch.equal(ops.attention_quant(q, step, 0.125, window, layer), want), window
    ops.check_error_flag()


# ---- lengths ------------------------------------------------------------------------------------------------------------

def test_lengths_on_the_device_past_the_hosts_bound_are_reported(ops, monkeypatch):
    """Each sequence brings as many tokens as the host planned for, but is longer on the device than the longest that the host
    knows of: the pages that were read back do not hold it."""
    from smolmoe_c99_b200.kernels import KernelError
    monkeypatch.setattr(ops, "quant_rows_tokens", 1)
    news, starts, slots = [60, 70], [66, 200], [0, 1]
    layer = make_layer("fp8", 2, 64, [600, 600], slots)
    fill(ops, layer, slots, [600, 600], 97)
    step = pack_step(slots, starts, [[0] * n for n in news], torch.device("cuda"))
    q = _randn((sum(news), 14, 64), 98).bfloat16()
    want = ops.attention_quant(q, step, 0.125, 0, layer)
    ops.check_error_flag()
    ends = step.seq_ends.clone()
    step.seq_ends += 256
    ops.attention_quant(q, step, 0.125, 0, layer)
    with pytest.raises(KernelError, match="attention_quant met|kv_quant_load met"):
        ops.check_error_flag()
    ops.kv_quant_load(step, layer, torch.bfloat16)
    with pytest.raises(KernelError, match="kv_quant_load met"):
        ops.check_error_flag()
    step.seq_ends.copy_(ends)
    assert torch.equal(ops.attention_quant(q, step, 0.125, 0, layer), want)
    ops.check_error_flag()


# ---- many sequences -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 128), (3, 1, 112), (9, 1, 128), (10, 1, 64)])
@pytest.mark.parametrize("n,cluster", [(1607, 0), (1608, 0), (1608, None), (2888, 0), (4096, None), (4096, 0), (4096, 8)])
def test_as_many_sequences_as_are_promised(ops, heads, kv_heads, hd, n, cluster, monkeypatch):
    """Single tokens, each sequence's numbers beside the tiles in shared memory."""
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    ends = [1 + (37 * i) % 90 for i in range(n)]
    slots = [n - 1 - i for i in range(n)]
    layer = make_layer("fp8", kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 99)
    q = _randn((n, heads, hd), 100).bfloat16()
    step = pack_step(slots, [e - 1 for e in ends], [[0]] * n, torch.device("cuda"))
    got = ops.attention_quant(q, step, hd ** -0.5, 0, layer)
    ops.check_error_flag()
    picked = [0, 1, 31, 32, 255, 256, 1023, 1024, n - 2, n - 1]
    want, room = row_by_row(layer, q[picked], [slots[i] for i in picked], [ends[i] - 1 for i in picked], [1] * len(picked), hd ** -0.5, 0)
    assert ((got[picked].double().cpu() - want).abs() <= room).all()
    # (the others against the plain kernel: both are rounded to bfloat16 once, and the weights of one of them)
    monkeypatch.setattr(ops, "use_fast_attention", False)
    plain = ops.attention_quant(q, step, hd ** -0.5, 0, layer).double()
    assert float((got.double() - plain).abs().max()) <= 2.0 ** -6 * float(plain.abs().max())


# ---- memory -------------------------------------------------------------------------------------------------------------

def _peak(call):
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("window,dtype", [(0, torch.bfloat16), (500, torch.bfloat16), (0, torch.float32)])
def test_what_a_mixed_step_reads_back_is_what_its_chunks_see(ops, window, dtype):
    """Many sequences that decode beside one that brings a portion onto a long one: the pages read back are those of the long
    one alone (within its window), not as many for each; in the 32-bit path those that each sequence holds."""
    n, heads, kv_heads, hd = 40, 8, 4, 128
    starts, news, slots = [9000] + [100 + i for i in range(n)], [300] + [1] * n, list(range(n + 1))
    ends = [s + k for s, k in zip(starts, news)]
    layer = make_layer("fp8", kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 101)
    q = _randn((sum(news), heads, hd), 102).to(dtype)
    step = pack_step(slots, starts, [[0] * k for k in news], torch.device("cuda"))
    page = 2 * kv_heads * 64 * hd * q.element_size()
    pages = -(-ends[0] // 64) if not window else -(-(window + news[0]) // 64) + 4
    if dtype == torch.float32:
        pages += sum(-(-e // 64) for e in ends[1:])
    room = pages * page + q.numel() * q.element_size() + (1 << 20)
    if dtype == torch.bfloat16:     # (what the two kernels keep their parts in)
        room += 4 * (ops.lib.sm_attention_chunk_workspace(hd, kv_heads, 10) + ops.lib.sm_attention_quant_workspace(hd, 2, kv_heads * (n + 1), 0))
    ops.attention_quant(q, step, hd ** -0.5, window, layer)
    assert _peak(lambda: ops.attention_quant(q, step, hd ** -0.5, window, layer)) <= room
    ops.check_error_flag()


# ---- pages read back ----------------------------------------------------------------------------------------------------

def test_slots_that_are_not_of_the_step_have_a_page_that_exists(ops):
    """kv_quant_load's page table has every slot of the cache's: those that the step does not name must not lead out of the pages
    that were read back."""
    layer = make_layer("int8", 2, 64, [100, 200, 70], [7, 2, 33])
    fill(ops, layer, [7, 2, 33], [100, 200, 70], 103)
    step = pack_step([33, 7], [69, 99], [[0], [0]], torch.device("cuda"))
    poison = torch.full((layer.page_table.shape[0], 2), 1 << 30, dtype=torch.int32, device="cuda")
    del poison                                   # (its memory is what the table is likely to get)
    back = ops.kv_quant_load(step, layer, torch.bfloat16)
    table = back.page_table.cpu()
    assert tuple(table.shape) == (35, 2) and int(table.min()) >= 0 and int(table.max()) < back.k_pool.shape[0]
    assert table[33].tolist() == [0, 1] and table[7].tolist() == [2, 3]
    ops.check_error_flag()


# ---- places, where the plain kernel attends ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 24)])
def test_places_outside_the_page_table_are_refused_by_the_plain_form(ops, dtype, hd):
    """Float queries and head sizes of no kernel of their own are attended by one that checks no place."""
    from smolmoe_c99_b200.kernels import KernelError
    layer = make_layer("fp8", 2, hd, [100, 128], [0, 1])
    fill(ops, layer, [0, 1], [100, 128], 104)
    q = _randn((2, 4, hd), 105).to(dtype)
    for slots, starts in (([0, layer.page_table.shape[0]], [99, 0]), ([0, 1], [99, 64 * layer.page_table.shape[1]])):
        with pytest.raises(KernelError, match="the page table"):
            ops.attention_quant(q, pack_step(slots, starts, [[0], [0]], torch.device("cuda")), 0.125, 0, layer)
    ops.attention_quant(q, pack_step([1, 0], [127, 99], [[0], [0]], torch.device("cuda")), 0.125, 0, layer)
    ops.check_error_flag()


# ---- long chunks in a window --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cluster", [None, 0, 1, 4])
@pytest.mark.parametrize("window", [1, 2, 31, 33, 64, 129, 400])
@pytest.mark.parametrize("heads,kv_heads,hd", [(3, 1, 32), (5, 5, 48), (9, 1, 96), (14, 2, 64)])
def test_long_chunks_in_a_window_straight_from_the_codes(ops, heads, kv_heads, hd, window, cluster, monkeypatch):
    """Each block of tokens attends over tiles of its own, at the sequence's start and around the tiles' edges."""
    monkeypatch.setattr(ops, "quant_cluster", cluster)
    monkeypatch.setattr(ops, "quant_rows_tokens", 1 << 20)
    starts, news, slots = [0, 61, 300], [150, 97, 40], [2, 0, 1]
    ends = [s + n for s, n in zip(starts, news)]
    layer = make_layer("int8", kv_heads, hd, ends, slots)
    fill(ops, layer, slots, ends, 106)
    q = _randn((sum(news), heads, hd), 107).bfloat16()
    check_rows(ops, layer, q, slots, starts, news, hd ** -0.5, window)


def test_the_work_of_a_long_chunk_in_a_window_grows_with_its_tokens(ops):
    """Head size 48 has no tcgen05 kernel. Four times the tokens take about four times as long, not sixteen times (on a GPU that
    both fill)."""
    def microseconds(n):
        layer = make_layer("fp8", 4, 48, [n], [0])
        fill(ops, layer, [0], [n], 108)
        q = _randn((n, 16, 48), 109).bfloat16()
        step = pack_step([0], [0], [[0] * n], torch.device("cuda"))
        best = float("inf")
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.attention_quant(q, step, 48 ** -0.5, 64, layer)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 1e3)
        return best
    short, long = microseconds(8192), microseconds(32768)
    assert long < 8 * short, f"{short:.0f} and {long:.0f} us"


# ---- the same slot twice ------------------------------------------------------------------------------------------------

def test_a_slot_twice_in_a_step(ops):
    """Two sequences of one slot that end at different positions. From the codes and through pages each is what it is alone; a page
    table by slot cannot tell them apart, so reading back and the plain form refuse."""
    from smolmoe_c99_b200.kernels import KernelError
    layer = make_layer("fp8", 2, 64, [300, 50], [1, 0])
    fill(ops, layer, [1, 0], [300, 50], 110)
    slots, starts = [1, 0, 1], [99, 49, 297]
    for news in ([1, 1, 1], [1, 1, 3]):
        step = pack_step(slots, starts, [[0] * n for n in news], torch.device("cuda"))
        q = _randn((sum(news), 4, 64), 111)
        for rows_tokens in (64, 1):
            ops.quant_rows_tokens = rows_tokens
            try:
                check_rows(ops, layer, q.bfloat16(), slots, starts, news, 0.125, 0)
            finally:
                ops.quant_rows_tokens = None
        with pytest.raises(KernelError, match="slot appears twice"):
            ops.attention_quant(q, step, 0.125, 0, layer)
        with pytest.raises(KernelError, match="slot appears twice"):
            ops.kv_quant_load(step, layer, torch.float32)
