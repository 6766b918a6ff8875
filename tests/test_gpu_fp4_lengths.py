"""Lengths of the 4-bit cache that a caller has set: one meaning in every call, made by the binding or by Python."""
import pytest
import torch

import operators_ref as R
from gaac_amd import FP4KVCache, _lib
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("python", [False, True])
def test_below_zero_is_empty_and_above_the_capacity_full(python, monkeypatch):
    require_gpu()
    if python: monkeypatch.setattr(_lib, "_calls", _lib._CtypesCalls())
    n_kv, L = 2, 64
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(L, n_kv, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    c = FP4KVCache(6, n_kv, L)
    for s in range(6): c.prefill(s, k, v)
    c.lens.copy_(torch.tensor([-40, 64, 2 ** 31 - 1, -2 ** 31, 65, 7], dtype=torch.int32))
    held = [0, 64, 64, 0, 64, 7]
    for s, n in enumerate(held):
        for got, x in zip(c.decompress(s), (k, v)):
            assert got.shape == (n, n_kv, D) and torch.equal(got.double().cpu(), R.stored(x[:n]))
    st = c.stats()
    assert st["tokens"] == sum(held) and st["bytes_used"] == sum(held) * n_kv * 136 and abs(st["ratio"] - 512 / 136) < 1e-9
    q, slots = torch.randn(6, 4, D, generator=g).to(torch.bfloat16).cuda(), torch.arange(6, dtype=torch.int32, device="cuda")
    for nsplit in (1, 2):
        out = c.attention(q, slots, D ** -0.5, nsplit=nsplit).double().cpu()
        for s, n in enumerate(held):
            ref, tol = R.attention(q[s], R.stored(k[:n]), R.stored(v[:n]), D ** -0.5)
            assert ((out[s] - ref).abs() <= tol).all()
    before = c.data.clone()
    c.append(slots, k[:6], v[:6])      # but for the last one: full, or of no length
    assert c.lens.tolist() == [-40, 64, 2 ** 31 - 1, -2 ** 31, 65, 8] and torch.equal(c.data[:5 * n_kv], before[:5 * n_kv])
    with pytest.raises(RuntimeError, match="token capacity, or its length was set below 0"): c.check_capacity()


def test_the_lengths_of_an_empty_cache_and_of_one_on_another_stream():
    require_gpu()
    c = FP4KVCache(2, 1, 64)
    assert c.stats()["tokens"] == 0 and c.decompress(1)[0].shape == (0, 1, D)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x = torch.ones(50, 1, D, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)      # longer than the host looks at the word before it waits for the stream
        c.prefill(1, x, x)
        k, v = c.decompress(1)
        assert torch.equal(k, x) and torch.equal(v, x)


def test_a_slot_named_twice_is_reported_as_that():
    """Whether it is full, has one place left or many: what the second row reports does not depend on when the first one has raised the length."""
    require_gpu()
    k = torch.ones(64, 1, D, dtype=torch.bfloat16, device="cuda")
    for held, bits, length in ((64, 3, 64), (63, 2, 64), (10, 2, 11)):
        for B in (2, 64):
            c = FP4KVCache(1, 1, 64)
            c.prefill(0, k[:held], k[:held])
            c.append(torch.zeros(B, dtype=torch.int32, device="cuda"), k[:B], k[:B])
            assert int(c.overflow) == bits and c.lens.tolist() == [length]
