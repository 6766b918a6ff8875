"""Rows beyond one launch, and offsets past 32 bits."""
import pytest
import torch

import fp8_ref as R
from gaac_amd import FP8Weight, fp8_linear, quantize_fp8, rms_norm_fp8, token_logprobs
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def gpu():
    require_gpu()
    yield
    torch.cuda.empty_cache()


def test_more_rows_than_a_launch_has():
    M = (1 << 20) + 37
    x = torch.zeros(M, 40, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 127, 128, 1 << 19, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, M - 1], device="cuda")
    x[at] = torch.randn(len(at), 40, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    v = quantize_fp8(x).dequantize()
    assert torch.equal(v[at].double().cpu(), R.stored(x[at])) and int((v != 0).any(1).sum()) == len(at)
    w = torch.ones(40, dtype=torch.bfloat16, device="cuda")
    rows, h = rms_norm_fp8(x, w, 1e-6, residual=x)
    y, _ = R.norm(x[at], w, 1e-6, x[at])
    got = rows.dequantize()
    assert ((got[at].double().cpu() - y).abs() <= R.half_step(y) * 1.001).all() and int((got != 0).any(1).sum()) == len(at) and torch.equal(h, x + x)


def test_offsets_past_32_bits():
    """5.4e9 bytes of rows in 8 bits, 10.7e9 of outputs."""
    M, K, N = 81920, 65536, 65536
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    at, cols = torch.tensor([0, 5000, 33000, 65535, 65536, M - 1], device="cuda"), torch.tensor([0, 1, 40000, N - 1], device="cuda")
    x[at] = torch.randn(len(at), K, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    rows = quantize_fp8(x)
    assert rows.data.numel() > 1 << 32
    del x
    w = torch.zeros(N, 256, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(rows.dequantize()[at].double().cpu(), R.stored(R_rows(at, K)))
    del rows
    x = torch.zeros(M, 256, dtype=torch.bfloat16, device="cuda")
    x[at], w[cols] = R_rows(at, 256, 2), R_rows(cols, 256, 3)
    out = fp8_linear(x, FP8Weight(w))
    assert out.numel() > 1 << 32
    y, tol = R.product(R.stored(x[at]), R.stored(w[cols]), torch.bfloat16)
    assert ((out[at][:, cols].double().cpu() - y).abs() <= tol).all()
    rest = torch.ones(M, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert not out[rest][:, cols].any() and not out[rest][:, 7].any()


def R_rows(at, K, seed=1):
    return torch.randn(len(at), K, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(torch.bfloat16)


def test_logits_past_32_bits():
    B, V = 40000, 128000
    x = torch.zeros(B, V, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 1 << 32
    at = torch.tensor([0, 20000, 33554, B - 1], device="cuda")
    x[at] = torch.randn(len(at), V, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(torch.bfloat16)
    tokens = torch.arange(B, device="cuda") * 3
    out = token_logprobs(x, tokens, top=3)
    value, rank, entropy, top_values, top_tokens, tol, tol_entropy = R.logprobs(x[at], tokens[at], 3)
    assert ((out.logprob[at].double().cpu() - value).abs() <= tol(value)).all() and torch.equal(out.rank[at].cpu(), rank) and torch.equal(out.top_tokens[at].cpu(), top_tokens)
    assert torch.equal(out.top_tokens[1], torch.arange(3, device="cuda")) and out.rank[100] == 300
