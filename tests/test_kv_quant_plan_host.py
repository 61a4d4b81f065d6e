"""How much of an 8-bit cache a step reads back, counted on the host."""
import random
from types import SimpleNamespace

import pytest
import torch

from smolmoe_c99_b200.engine.batch import pack_step
from smolmoe_c99_b200.kernels import KernelError, Ops


@pytest.mark.parametrize("window", [0, 1, 64, 65, 300])
def test_pages_that_are_read_back(window, monkeypatch):
    """Against a count position by position; a captured step's bound holds for every start that its span allows."""
    rng = random.Random(window)
    layer, capturing = SimpleNamespace(table_stride=20, pages=60), False
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    for _ in range(60):
        starts, news = zip(*[(rng.choice([0, 1, 63, 64, 127, 128, 129, rng.randrange(1000)]), rng.choice([1, 2, 65, 200])) for _ in range(rng.randint(1, 6))])
        step = pack_step(list(range(len(starts))), list(starts), [[0] * n for n in news], torch.device("cpu"))
        skip = rng.choice([0, 1, 64])
        reading = [(s, n) for s, n in zip(starts, news) if n > skip]
        if not reading:
            continue
        taken = []
        for s, n in reading:
            seen = {p // 128 for t in range(s, s + n) for p in range(max(0, t - window + 1) if window else 0, t + 1)}
            taken.append(sum(1 for page in range(-(-(s + n) // 64)) if page // 2 >= min(seen)))
        capturing = False
        most, room, seqs, pages = Ops._pages_read(step, layer, SimpleNamespace(exclusive=False), skip, window)
        assert (most, room, seqs, pages) == (-(-max(s + n for s, n in zip(starts, news)) // 64), sum(taken), len(taken), max(taken))
        capturing = True
        step.max_seq_len = 1280
        for exclusive in (False, True):
            most, room, seqs, pages = Ops._pages_read(step, layer, SimpleNamespace(exclusive=exclusive), skip, window)
            assert most == 20 and seqs == len(taken) and pages >= max(taken)
            assert room >= sum(taken) if not exclusive else room == min(60, room)
        step.seq_starts, capturing = None, False          # (a decode step's graph knows no starts)
        assert Ops._pages_read(step, layer, SimpleNamespace(exclusive=False), skip, window)[1] >= sum(taken)


@pytest.mark.parametrize("slots,starts,message", [([0, 5], [0, 9], "slots 0 to 5: the page table has 5"), ([-1, 2], [0, 9], "slots -1 to 2"),
                                                  ([0, 4], [3, 126], "129 positions: the page table holds 128")])
def test_places_outside_the_page_table_are_refused_where_no_kernel_would(slots, starts, message):
    step = pack_step(slots, starts, [[0, 0], [0, 0, 0]], torch.device("cpu"))
    with pytest.raises(KernelError, match=message):
        Ops._check_places(step, SimpleNamespace(slots=5, table_stride=2))


def test_places_inside_the_page_table_are_not_refused():
    layer = SimpleNamespace(slots=5, table_stride=2)
    Ops._check_places(pack_step([0, 4], [3, 125], [[0, 0], [0, 0, 0]], torch.device("cpu")), layer)
    Ops._check_places(SimpleNamespace(slots=[], seq_starts=None), layer)


def test_each_bounded_wait_of_the_chunk_kernel_has_a_code_of_its_own():
    import os
    import re

    import smolmoe_c99_b200
    with open(os.path.join(os.path.dirname(smolmoe_c99_b200.__file__), "csrc", "attention_chunk_tc.cu")) as f:
        codes = [int(c) for c in re.findall(r"fail\((\d+)\)", f.read())]
    assert len(codes) >= 10 and len(set(codes)) == len(codes) and all(41 <= c <= 52 for c in codes), sorted(codes)


def test_a_slot_twice_is_refused_where_pages_are_found_by_slot():
    with pytest.raises(KernelError, match="slot appears twice"):
        Ops._check_slots_once(pack_step([1, 0, 1], [3, 0, 9], [[0], [0], [0]], torch.device("cpu")))
    Ops._check_slots_once(pack_step([1, 0, 2], [3, 0, 9], [[0], [0], [0]], torch.device("cpu")))
