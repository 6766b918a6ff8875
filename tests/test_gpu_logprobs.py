"""Log probabilities, ranks, entropy and alternatives against their definition in 64 bits."""
import pytest
import torch

import fp8_ref as R
from gaac_amd import token_logprobs
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def gpu(): require_gpu()


def check(logits, tokens, top):
    out = token_logprobs(logits, tokens, top=top)
    value, rank, entropy, top_values, top_tokens, tol, tol_entropy = R.logprobs(logits, tokens, top)

    def within(a, y, t):
        a = a.double().cpu()
        assert a.shape == y.shape and torch.equal(a.isnan(), y.isnan()) and torch.equal(a[a.isinf()], y[y.isinf()]) and torch.equal(a.isinf(), y.isinf())
        fine = a.isfinite()
        assert ((a - y).abs() <= t)[fine].all(), (a - y)[fine].abs().max()
    within(out.logprob, value, tol(value))
    within(out.entropy, entropy, tol_entropy)
    assert out.rank.dtype == torch.int64 and torch.equal(out.rank.cpu(), rank)
    if top == 0: assert out.top_logprobs is None and out.top_tokens is None
    else:
        assert torch.equal(out.top_tokens.cpu(), top_tokens)
        within(out.top_logprobs, top_values, tol(top_values))


def logits_of(B, V, seed=0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * 2.5
    x[torch.arange(B)[:, None], torch.randint(0, V, (B, 20), generator=g)] += torch.rand(B, 20, generator=g) * 10
    return x.to(dtype).cuda(), torch.randint(0, V, (B,), generator=g).cuda()


@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 7), (2, 64), (5, 1000), (4, 8191), (2, 8192), (3, 8193), (2, 16385), (4, 128256), (1, 262144)])
def test_rows(B, V, top, dtype):
    if top > V: pytest.skip("more alternatives than logits")
    check(*logits_of(B, V, seed=B + V, dtype=dtype), top)


@pytest.mark.parametrize("V", [50, 3000, 20000])
@pytest.mark.parametrize("top", [0, 3, 33])
def test_rows_of_every_kind(V, top):
    x, tokens = logits_of(16, V, seed=V, dtype=FP32)
    x[0] = -torch.inf
    x[1] = torch.nan
    x[2, ::2] = -torch.inf
    x[3, 5], x[3, V - 1] = torch.inf, torch.inf
    x[4, 1::3] = torch.nan
    x[5] = 1.5                                             # all alike: by index
    x[6] = torch.arange(V, device="cuda") / 64.0           # rising
    x[7] = -torch.arange(V, device="cuda") / 64.0          # falling
    x[8, :] = -torch.inf
    x[8, V // 2] = -3.0                                    # one token only
    x[9] = torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, -0.0)      # 0 and -0 are alike
    x[10] = torch.randint(0, 3, (V,), generator=torch.Generator().manual_seed(1)).float().cuda()      # many ties
    x[11] *= 1e30
    x[12] = torch.finfo(FP32).min                          # the type's lowest, not -inf
    x[12, 7] = 0
    x[13, 0], x[13, 1:] = 80.0, x[13, 1:] - 40
    tokens[:4] = torch.tensor([0, V - 1, 1, 5])
    tokens[14], tokens[15] = -1, V
    check(x, tokens, min(top, V))
    check(x.to(BF), tokens.roll(3), min(top, V))


@pytest.mark.parametrize("dtype", [BF, FP32])
def test_strides(dtype):
    wide, tokens = logits_of(12, 9001, seed=5, dtype=dtype)
    for x in (wide[:, :9000], wide[:, 1:], wide[:, 3:8200], wide[::2], wide.flip(0), wide[:1].expand(12, 9001), wide[:, ::3]):
        check(x, tokens[:x.shape[0]] % x.shape[1], 10)
    check(wide, torch.stack([tokens, tokens], 1)[:, 0], 2)
    out = token_logprobs(wide[:0], tokens[:0], top=3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0,), (0, 3), (0, 3)]


def test_the_same_each_time():
    x, tokens = logits_of(50, 30000, seed=7)
    first = token_logprobs(x, tokens, top=20)
    for _ in range(3):
        for a, b in zip(first, token_logprobs(x, tokens, top=20)): assert torch.equal(a, b)
