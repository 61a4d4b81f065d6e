"""The engine with its cache in 8 bits: every way of cutting the requests into steps, against itself (in the 32-bit path the
bits are the same) and against the plain implementation with its keys and values rounded to the cache."""
import pytest
import torch

import plain_model
import replay
from test_gpu_kv_quant import plain_rows
from tiny import TINY, random_tokens

pytestmark = pytest.mark.gpu

LENGTHS = {"A": [5, 17, 64, 65, 100], "B": [1, 23, 41, 96], "C": [3, 99, 130, 300], "D": [2, 127, 129, 420], "E": [5, 130, 260]}


def _requests(name, seed=70):
    return {f"r{i}": random_tokens(n, TINY[name]["vocab_size"], seed + i) for i, n in enumerate(LENGTHS[name])}


def _engine(folder, dtype, fmt, **kw):
    from smolmoe_c99_b200.engine.engine import Engine
    return Engine(folder, dtype, max_tokens=2048, kv_dtype=fmt, **kw)


def _cuts(engine, requests):
    ids = list(requests)
    heads = {r: max(1, len(requests[r]) * 2 // 3) for r in ids}
    yield "whole", replay.whole(engine, requests)
    yield "tail", replay.tail_decoded(engine, requests, 9)
    yield "batched", replay.batched(engine, [{r: requests[r] for r in ids[:2]}, {r: requests[r] for r in ids[2:]}], heads)
    yield "portions", replay.portions(engine, requests, 37, 3)
    yield "portions again", replay.portions(engine, requests, 37, 3)       # (shapes seen before are replayed graphs)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_every_cut_gives_the_same_bits_in_32_bits(model_dirs, name, fmt):
    engine = _engine(model_dirs[name], "float32", fmt)
    requests = _requests(name)
    want = None
    for cut, got in _cuts(engine, requests):
        want = want or got
        for r in requests:
            assert torch.equal(got[r], want[r]), f"{cut} {r}: {float((got[r] - want[r]).abs().max()):.3g}"
    engine.check_status()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E"])
def test_logits_against_the_plain_implementation(model_dirs, name, fmt, dtype, monkeypatch):
    """What the rounding of keys and values does to the logits, D, comes from N values each off by up to half a step.
    Where the engine's own value is on the other side of a border than the plain one, a value is off by a whole step; in
    the 32-bit path that is about one value in 10,000 or none, so the sum moves by a small part of D (1 / (0.29 sqrt(N)),
    N in the thousands); in bfloat16 up to 2^-9 / 2^-4 of all values, sqrt(1 / 32) / 0.29 = 0.6 of D, twice that for the
    worst of many logits. On top of the bounds of the engine without an 8-bit cache (compare.py)."""
    requests = _requests(name)
    rounded = dtype == "bfloat16"
    without = {r: plain_model.forward(model_dirs[name], t, round_like_bf16_engine=rounded) for r, t in requests.items()}
    attend = plain_model.attend
    monkeypatch.setattr(plain_model, "attend", lambda q, k, v, *rest: attend(
        q, plain_rows(k, fmt).to(k.dtype), plain_rows(v, fmt).to(v.dtype), *rest))
    want = {r: plain_model.forward(model_dirs[name], t, round_like_bf16_engine=rounded) for r, t in requests.items()}
    engine = _engine(model_dirs[name], dtype, fmt)
    part, base = (0.25, 5e-6) if dtype == "float32" else (1.2, 1e-2)
    moved = max(float((want[r] - without[r]).abs().max() / want[r].abs().max()) for r in requests)
    assert moved > 1e-4
    for cut, got in _cuts(engine, requests):
        for r in requests:
            off = float((got[r] - want[r]).abs().max() / want[r].abs().max())
            assert off <= part * moved + base, f"{cut} {r}: {off:.3g}, the cache's rounding moves the logits by {moved:.3g}"


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("name", ["B", "C", "D"])
def test_the_first_layers_cache_is_the_other_caches_rounded(model_dirs, name, fmt):
    """Keys and values of the first layer do not depend on any attention: the 8-bit cache holds what the bfloat16 cache
    holds, rounded, position by position, after prompts, portions and single tokens."""
    from smolmoe_c99_b200.engine.engine import Engine
    toks = _requests(name)["r3"] if "r3" in _requests(name) else random_tokens(90, TINY[name]["vocab_size"], 1)
    other = random_tokens(30, TINY[name]["vocab_size"], 2)
    views = []
    for kind in (None, fmt):
        engine = Engine(model_dirs[name], "bfloat16", max_tokens=2048, kv_dtype=kind)
        a, b = engine.open_sequence(), engine.open_sequence()
        engine.step([a, b], [toks[:40], other[:7]])
        engine.step([b, a], [other[7:20], toks[40:41]])
        for i in range(41, len(toks) - 1, 2):
            engine.step([a], [toks[i:i + 2]])
        engine.step([b, a], [other[20:21], toks[-1:]])
        engine.step([b], [other[21:22]])
        views.append((engine, {a: engine.length(a), b: engine.length(b)}))
    (e0, lengths), (e1, _) = views
    from test_gpu_kv_quant import held
    full, packed = e0.cache.run_view(0), e1.cache.run_view(0)
    assert full.ring == 0
    for slot, n in lengths.items():
        for which in "kv":
            pool = full.k_pool if which == "k" else full.v_pool
            pages = full.page_table[slot, :-(-n // 64)].long()
            rows = pool[pages].permute(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3])[:n]
            assert torch.equal(held(packed, which, slot, n), plain_rows(rows, fmt)), (slot, which)


def test_a_layer_that_reads_anothers_8_bit_cache(tmp_path):
    from smolmoe_c99_b200.config import config_from_json, register_architecture
    from smolmoe_c99_b200.engine.engine import Engine
    from smolmoe_c99_b200.weights import write_random_model
    from test_gpu_parts import SharedOrderConfig
    register_architecture("SharedOrderForCausalLM", SharedOrderConfig)
    folder = write_random_model(config_from_json(dict(TINY["A"], architectures=["SharedOrderForCausalLM"])), str(tmp_path / "m"), 3)
    requests = {f"r{i}": random_tokens(n, 256, 60 + i) for i, n in enumerate([3, 40, 77])}
    engine = Engine(folder, "float32", max_tokens=1024, kv_dtype="int8")
    assert len(engine.cache.groups) == 1 and engine.cache.groups[0].n_layers == 3
    want = None
    for cut, got in _cuts(engine, requests):
        want = want or got
        assert all(torch.equal(got[r], want[r]) for r in requests), cut
    # bfloat16 against the 32-bit engine, by the bound of the plain comparison above: what the cache's rounding moves the logits
    # by is measured between the 32-bit engines with and without it
    without = replay.whole(Engine(folder, "float32", max_tokens=1024), requests)
    moved = max(float((want[r] - without[r]).abs().max() / want[r].abs().max()) for r in requests)
    bfloat = Engine(folder, "bfloat16", max_tokens=1024, kv_dtype="int8")
    for cut, got in _cuts(bfloat, requests):
        for r in requests:
            off = float((got[r] - want[r]).abs().max() / want[r].abs().max())
            assert off <= 1.2 * moved + 1e-2, f"{cut} {r}: {off:.3g}, the cache's rounding moves the logits by {moved:.3g}"


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_generation(model_dirs, fmt, dtype):
    """Batches of unequal prompts through the Python entry point; in the 32-bit path a request's tokens do not depend on
    what it is batched with, and the plain kernels give what the fast ones give."""
    from smolmoe_c99_b200 import Model
    prompts = [random_tokens(n, TINY["D"]["vocab_size"], 80 + n) for n in (3, 64, 90, 200, 17)]
    model = Model.from_folder(model_dirs["D"], dtype, context=512, batch=3, kv_dtype=fmt)
    got = model.generate(prompts, tokens=70, stop_ids=())
    assert [len(t) for t in got] == [70] * 5
    if dtype == "float32":
        alone = Model.from_folder(model_dirs["D"], dtype, context=512, batch=1, kv_dtype=fmt, step_tokens=50)
        assert alone.generate(prompts, tokens=70, stop_ids=()) == got
        plain = Model.from_folder(model_dirs["D"], dtype, context=512, batch=5, kv_dtype=fmt, kernels="plain")
        assert plain.generate(prompts, tokens=70, stop_ids=()) == got
    assert model.engine.cache.bytes_per_token() == 2 * 2 * 3 * 65


def test_a_sequence_cut_back_and_fed_again(model_dirs):
    engine = _engine(model_dirs["C"], "float32", "fp8")     # (windowed layers keep every position: cutting back is possible)
    toks = random_tokens(150, TINY["C"]["vocab_size"], 5)
    slot = engine.open_sequence()
    want = engine.step([slot], [toks], [list(range(150))]).cpu()
    engine.cache.truncate(slot, 60)
    got = engine.step([slot], [toks[60:]], [list(range(90))]).cpu()
    assert torch.equal(got, want[60:])


def test_the_command_line(model_dirs, capsys):
    import json
    from smolmoe_c99_b200.engine import cli
    assert cli.main([model_dirs["A"], "--prompt", "5 17 3", "--tokens", "4", "--kv-dtype", "fp8", "--stop-ids", ""]) == 0
    said = capsys.readouterr()
    assert len(said.out.split()) == 4
    stats = json.loads(said.err.strip().splitlines()[-1])
    assert stats["kv_dtype"] == "fp8" and stats["kv_bytes"] == 2 * 2 * 2 * 17 * 1024


def test_the_fused_decode_option_leaves_an_8_bit_cache_to_its_own_kernels(model_dirs):
    """The one-kernel decode step reads caches of the compute type alone: with the option on the bits are the same."""
    from smolmoe_c99_b200.kernels import get_ops
    ops = get_ops()
    requests = _requests("A")
    want = replay.tail_decoded(_engine(model_dirs["A"], "bfloat16", "fp8"), requests, 9)
    before = ops.use_fused_decode
    ops.use_fused_decode = True
    try:
        got = replay.tail_decoded(_engine(model_dirs["A"], "bfloat16", "fp8"), requests, 9)
    finally:
        ops.use_fused_decode = before
    assert all(torch.equal(got[r], want[r]) for r in requests)
