"""Batches of the 4-bit cache whose rows have more than 2^31 tiles between them: the plan of the splits counts tiles in 32 bits."""
import pytest
import torch

from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
D = 128


def test_rows_of_more_than_two_to_the_31_tiles():
    """2048 rows that name one slot of 2^25 tokens, 2^31 tiles in all (the sum of the tiles used to pass 32 bits, and with it the place of a row's tiles).  Keys are 0 and values 1, so
    that every sum is exact and every output 1."""
    from gaac_amd import FP4KVCache
    require_gpu()
    L, B = 1 << 25, 2048
    c = FP4KVCache(1, 1, L)
    k, v = torch.zeros(1, 1, D, dtype=torch.bfloat16, device="cuda"), torch.ones(1, 1, D, dtype=torch.bfloat16, device="cuda")
    c.prefill(0, k.expand(L, 1, D), v.expand(L, 1, D))
    q, slots = torch.ones(B, 1, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    out = c.attention(q, slots, D ** -0.5, nsplit=2)
    assert (out == 1).all()
    c.lens.fill_(100)      # the same batch over a short row, against one row by itself
    q = torch.randn(B, 1, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    x = torch.randn(100, 1, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    c.prefill(0, x, x.flip(0).contiguous())
    out = c.attention(q, slots, D ** -0.5, nsplit=2)
    for b in (0, 1, 1023, 2047): assert torch.equal(out[b:b + 1], c.attention(q[b:b + 1], slots[:1], D ** -0.5, nsplit=1))
