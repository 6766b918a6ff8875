"""What a 4-bit cache holds in memory, and what of it is saved."""
import pickle

import torch

from gaac_amd import FP4KVCache


def tensors(x, seen):
    if isinstance(x, torch.Tensor): seen[x.untyped_storage().data_ptr()] = x.untyped_storage().nbytes()
    elif isinstance(x, dict):
        for y in x.values(): tensors(y, seen)
    elif isinstance(x, (list, tuple)):
        for y in x: tensors(y, seen)
    return sum(seen.values())


def test_a_cache_holds_what_its_slots_are_said_to_take():
    for n_slots, n_kv, capacity in ((3, 8, 256), (1, 4, 100), (5, 1, 33), (2, 8, 4096)):
        c = FP4KVCache(n_slots, n_kv, capacity, device="cpu")
        assert tensors(vars(c), {}) == n_slots * FP4KVCache.bytes_per_slot(n_kv, capacity) + 4      # and the word of check_capacity


def test_a_budget_is_kept():
    from gaac_amd.serving import Attention, allocate_fp4_cache
    per_slot = FP4KVCache.bytes_per_slot(8, 256)
    layers = [Attention(32, 128, 0.1, 8) for _ in range(3)]
    num, caches = allocate_fp4_cache(layers, 3 * 7 * per_slot + per_slot, 8, 256, 100, device="cpu")
    assert num == 7 and sum(tensors(vars(c), {}) for c in caches) <= 3 * 7 * (per_slot + 4)


def test_saved_caches_have_no_counters():
    """Counters are of the streams and graphs of one process; caches saved while they were attributes of another form are read as well."""
    c = FP4KVCache(2, 4, 64, device="cpu")
    c.lens[1] = 5
    c._tickets[0] = torch.ones(64, dtype=torch.int32)
    c._given.append(torch.ones(64, dtype=torch.int32))
    d = pickle.loads(pickle.dumps(c))
    assert d._tickets == {} and d._captured == 0 and d.lens.tolist() == [0, 5] and torch.equal(d.data, c.data) and c._captured == 1
    old = FP4KVCache.__new__(FP4KVCache)
    old.__setstate__(dict(n_slots=2, n_kv=4, tiles=2, cap=64, H=8, data=c.data, lens=c.lens, overflow=c.overflow, _tickets={0: c.lens}, _spare=torch.ones(64, 256, dtype=torch.int32), _captured=3))
    assert old._tickets == {} and old._captured == 0 and not hasattr(old, "_spare") and old.cap == 64


def test_attention_on_the_host_is_refused_by_name_with_splits_too():
    import pytest
    c = FP4KVCache(2, 4, 4096, device="cpu")
    for nsplit in (1, 3):
        with pytest.raises(RuntimeError, match="no CPU path"): c.attention(torch.zeros(1, 4, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), 1.0, nsplit=nsplit)


def test_stats_of_lengths_that_a_caller_set():
    c = FP4KVCache(4, 2, 64, device="cpu")
    c.lens.copy_(torch.tensor([-40, 64, 2 ** 31 - 1, 7], dtype=torch.int32))
    assert c.stats()["tokens"] == 135 and c.stats()["bytes_used"] == 135 * 2 * 136


def test_the_length_for_the_host_is_refused_without_its_words():
    import pytest
    from gaac_amd import _lib
    for args in ((None, 2, 16, None), (16, 2, None, None), (16, 0, 16, None), (16, 1 << 26, 16, None)):
        with pytest.raises(RuntimeError, match="gaac_fp4_length failed .*bad arguments"): _lib.call("gaac_fp4_length", *args)
