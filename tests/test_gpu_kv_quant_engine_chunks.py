"""The engine over an 8-bit cache where portions of prompts attend through pages read back and the tcgen05 kernel, eagerly and
captured: which way a portion takes is set by the number of its tokens, here from two tokens on."""
import pytest
import torch

import replay
from compare import check_logits
from tiny import TINY, random_tokens

pytestmark = pytest.mark.gpu

WINDOW = dict(use_sliding_window=True, sliding_window=150, max_window_layers=0)
CONFIGS = {"D": TINY["D"], "E": TINY["E"], "D in a window": dict(TINY["D"], **WINDOW), "E in a window": dict(TINY["E"], **WINDOW)}


@pytest.fixture
def pages_from_two_tokens(monkeypatch):
    """Routes chunks through pages (or, given a large number, none) and counts the calls that read pages back."""
    from smolmoe_c99_b200.kernels import Ops, get_ops
    calls, pages_read = [], Ops._pages_read
    monkeypatch.setattr(Ops, "_pages_read", staticmethod(lambda *args: calls.append(args[3]) or pages_read(*args)))

    def route(tokens):
        monkeypatch.setattr(get_ops(), "quant_rows_tokens", tokens)
        calls.clear()
        return calls
    return route


def _folder(tmp_path, config, layers):
    from smolmoe_c99_b200.config import config_from_json
    from smolmoe_c99_b200.weights import write_random_model
    return write_random_model(config_from_json(dict(config, num_hidden_layers=layers)), str(tmp_path / "m"), 11)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("name", list(CONFIGS))
def test_portions_through_pages_against_portions_from_the_codes(tmp_path, pages_from_two_tokens, name, fmt):
    """One layer, so that what the cache holds does not depend on any attention: the same steps, attended in both ways, differ by
    the rounding of weights and outputs alone."""
    from smolmoe_c99_b200.engine.engine import Engine
    folder = _folder(tmp_path, CONFIGS[name], 1)
    vocab = CONFIGS[name]["vocab_size"]
    first = {f"r{i}": random_tokens(n, vocab, 120 + i) for i, n in enumerate([90, 140])}
    second = {f"s{i}": random_tokens(n, vocab, 130 + i) for i, n in enumerate([400, 333, 70])}
    results = []
    for tokens in (1 << 20, 1):
        calls = pages_from_two_tokens(tokens)
        engine = Engine(folder, "bfloat16", max_tokens=4096, kv_dtype=fmt)
        cuts = {"portions": lambda: replay.portions(engine, second, 64), "portions again": lambda: replay.portions(engine, second, 64),
                "odd portions": lambda: replay.portions(engine, second, 149, 2),
                "joined": lambda: replay.joined(engine, first, second, {"r0": 60, "r1": 60, "s0": 390, "s1": 200, "s2": 60}, 5, 100)}
        results.append({cut: run() for cut, run in cuts.items()})
        engine.check_status()
        assert (len(calls) > 0) == (tokens == 1)
    for cut, want in results[0].items():
        check_logits(results[1][cut], want, "bfloat16", f"{name} {fmt} {cut}")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", list(CONFIGS))
def test_captured_portions_give_the_bits_of_eager_ones(tmp_path, pages_from_two_tokens, name, dtype):
    """A captured step is replayed at other starts than it was captured at; its span passes the sequence's length, and the room it
    reads back into is a bound."""
    from smolmoe_c99_b200.engine.engine import Engine
    folder = _folder(tmp_path, CONFIGS[name], 2)
    requests = {f"r{i}": random_tokens(n, CONFIGS[name]["vocab_size"], 140 + i) for i, n in enumerate([64 * 7, 64 * 13])}
    calls = pages_from_two_tokens(1)
    eager = Engine(folder, dtype, max_tokens=1024, kv_dtype="fp8", use_graphs=False)
    want = replay.portions(eager, requests, 64)
    assert calls
    captured = Engine(folder, dtype, max_tokens=1024, kv_dtype="fp8")
    for again in range(2):
        got = replay.portions(captured, requests, 64)
        assert all(torch.equal(got[r], want[r]) for r in requests), again
    assert len(captured._step_graphs) > 1
    captured.check_status()
    eager.check_status()
