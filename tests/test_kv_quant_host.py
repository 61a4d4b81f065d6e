"""The host's share of the 8-bit cache: what a cache of each kind holds, and what the kernels' faces refuse."""
import dataclasses

import pytest
import torch

from smolmoe_c99_b200.cache import LayerCache, SequenceCache
from smolmoe_c99_b200.kernels import KernelError, Ops
from smolmoe_c99_b200.parts import KVNeed


def _cache(**kw):
    needs = [KVNeed(2, 64), KVNeed(2, 64, 100), 0]
    return SequenceCache(needs, max_tokens=640, max_slots=4, max_seq_len=512, dtype=torch.bfloat16, device="cpu", **kw)


@pytest.mark.parametrize("kv_dtype,dtype", [("fp8", torch.float8_e4m3fn), ("int8", torch.int8)])
def test_what_an_8_bit_cache_holds(kv_dtype, dtype):
    cache = _cache(kv_dtype=kv_dtype)
    for run in (0, 1, 2):
        view = cache.run_view(run)
        assert view.k_pool.dtype == view.v_pool.dtype == dtype and tuple(view.k_pool.shape) == (10, 2, 64, 64)
        assert view.k_scale.dtype == torch.uint8 and tuple(view.k_scale.shape) == tuple(view.v_scale.shape) == (10, 2, 64)
        assert not view.k_pool.float().any()
    assert cache.run_view(2).k_scale.data_ptr() == cache.run_view(0).k_scale.data_ptr()    # (a run that reads another's)
    assert cache.run_view(1).ring == 0 and cache.run_view(1).window == 100                 # every position is kept
    assert cache.bytes_per_token() == 2 * 2 * 2 * (64 + 1)
    slot = cache.alloc_slot()
    cache.reserve({slot: 300})
    cache.advance({slot: 300})
    assert [len(g.slot_pages[slot]) for g in cache.groups] == [5, 5]
    cache.truncate(slot, 120)        # (possible in a windowed layer too: nothing was dropped)
    assert cache.length(slot) == 120


def test_a_cache_of_the_compute_type_is_what_it_was():
    cache = _cache()
    view = cache.run_view(1)
    assert view.k_pool.dtype == torch.bfloat16 and view.k_scale is None and view.ring == 128
    assert cache.bytes_per_token() == 2 * 2 * 2 * 64 * 2


def test_an_unknown_kind_is_refused():
    with pytest.raises(ValueError, match="kv_dtype must be one of fp8, int8"):
        _cache(kv_dtype="fp4")


@pytest.mark.parametrize("change,message", [
    (dict(k_scale=None), "8-bit key/value cache is needed"),
    (dict(kind="state"), "8-bit key/value cache is needed"),
    (dict(k_pool=torch.zeros(3, 2, 64, 64)), "float8_e4m3fn or int8"),
    (dict(v_pool=torch.zeros(3, 2, 64, 64, dtype=torch.float8_e4m3fn)), "float8_e4m3fn or int8"),
    (dict(v_pool=torch.zeros(4, 2, 64, 64, dtype=torch.int8)), "pools of an 8-bit cache are"),
    (dict(k_scale=torch.zeros(3, 2, 32, dtype=torch.uint8)), "pools of an 8-bit cache are"),
    (dict(k_scale=torch.zeros(3, 2, 64, dtype=torch.int8)), "uint8"),
    (dict(ring=128), "no ring"),
    (dict(page_table=torch.zeros(4, 8, dtype=torch.int64)), "int32"),
    (dict(page_table=torch.zeros(8, 4, dtype=torch.int32).T), "contiguous"),
])
def test_refused_caches(change, message):
    good = LayerCache("kv", torch.zeros(3, 2, 64, 64, dtype=torch.int8), torch.zeros(3, 2, 64, 64, dtype=torch.int8),
                      torch.zeros(4, 8, dtype=torch.int32), 0, None, k_scale=torch.zeros(3, 2, 64, dtype=torch.uint8),
                      v_scale=torch.zeros(3, 2, 64, dtype=torch.uint8))
    with pytest.raises(KernelError, match=message):
        Ops._quant_cache(None, dataclasses.replace(good, **change))


def test_the_command_line_names_the_kinds(capsys):
    from smolmoe_c99_b200.engine import cli
    with pytest.raises(SystemExit):
        cli.main(["x", "--kv-dtype", "fp4"])
    assert "fp8" in capsys.readouterr().err
