"""Refusals of rows and weights in 8 bits, their products and log probabilities, without a GPU: every call that cannot be made raises before anything is launched."""
import pytest
import torch
from torch.autograd import forward_ad

from gaac_amd import FP8Rows, FP8Weight, _lib, fp8_gated, fp8_linear, quantize_fp8, rms_norm_fp8, token_logprobs
from gaac_amd.fp8 import _memory
from gaac_amd.sampling import logprobs_work_bytes

X = torch.zeros(5, 256)


def weight(N=64, K=256, gated=False):
    """An FP8Weight without a device."""
    w = FP8Weight.__new__(FP8Weight)
    w.N, w.K, w.gated = N, K, gated
    w.data, w.exps = _memory(-(-N // 16) * 16 * (1 + gated), K, "cpu")
    return w


def test_sizes():
    data, exps = _memory(32, 700, "cpu")
    assert data.numel() == 32 * 768 and exps.numel() == 32 * 8
    assert weight(17, 129, True).nbytes == 64 * 256 + 64 * 4
    assert [logprobs_work_bytes(*x) for x in ((4, 8192, 20), (4, 8193, 20), (1, 128256, 0))] == [0, 4 * 2 * 176, 16 * 16]


def test_rows_that_are_refused():
    for call in (quantize_fp8, FP8Weight, lambda x: rms_norm_fp8(x, torch.ones(256))):
        for bad in (X.double(), X[0], X[None], X[:, :0], X.int()):
            with pytest.raises(RuntimeError, match=r"expects rows bf16, fp16 or fp32 \[M, K\]"): call(bad)
    with pytest.raises(RuntimeError, match="K up to 65536"): quantize_fp8(torch.zeros(1, 65537))
    with pytest.raises(RuntimeError, match="K up to 32768"): rms_norm_fp8(torch.zeros(1, 32769), torch.ones(32769))
    with pytest.raises(RuntimeError, match="2\\^24 rows"): quantize_fp8(torch.zeros(1, 8).expand((1 << 24) + 1, 8))
    for w in (torch.ones(256).half(), torch.ones(255), torch.ones(1, 256)):
        with pytest.raises(RuntimeError, match="rms_norm_fp8 expects weight"): rms_norm_fp8(X, w)
    for r in (X.half(), X[:4], X[:, :128], X[0]):
        with pytest.raises(RuntimeError, match="rms_norm_fp8 expects residual"): rms_norm_fp8(X, torch.ones(256), residual=r)
    with pytest.raises(RuntimeError, match="1 to 2\\^22 rows"): FP8Weight(X[:0])
    with pytest.raises(RuntimeError, match="1 to 2\\^22 rows"): FP8Weight(torch.zeros(1, 8).expand((1 << 22) + 1, 8))
    with pytest.raises(RuntimeError, match="of one shape"): FP8Weight(X, X[:4])
    for call in (lambda: quantize_fp8(X), lambda: FP8Weight(X), lambda: FP8Weight(X, X), lambda: rms_norm_fp8(X, torch.ones(256)), lambda: rms_norm_fp8(X, torch.ones(256), residual=X)):
        with pytest.raises(RuntimeError, match="no CPU path"): call()


def test_products_that_are_refused():
    w, pair = weight(), weight(gated=True)
    rows = FP8Rows(*_memory(16, 256, "cpu"), (5, 256))
    for x in (X, rows):
        with pytest.raises(RuntimeError, match="FP8Weight of one weight"): fp8_linear(x, pair)
        with pytest.raises(RuntimeError, match="FP8Weight of a gate and an up projection"): fp8_gated(x, w)
        with pytest.raises(RuntimeError, match="FP8Weight of one weight, got Tensor"): fp8_linear(x, X)
        with pytest.raises(RuntimeError, match="makes bf16, fp16 or fp32"): fp8_linear(x, w, out_dtype=torch.float64)
        with pytest.raises(RuntimeError, match="the weight's 128 inputs"): fp8_linear(x, weight(K=128))
        with pytest.raises(RuntimeError, match="in bf16 into 8 bits"): fp8_gated(x, pair, out_dtype=torch.float32, quantize=True)
        for call in (lambda: fp8_linear(x, w), lambda: fp8_gated(x, pair), lambda: fp8_gated(x, pair, quantize=True)):
            with pytest.raises(RuntimeError, match="no CPU path"): call()
    for bad in (X.double(), X[0], X[None], X[0, 0]):
        with pytest.raises(RuntimeError, match="expects rows bf16"): fp8_linear(bad, w, out_dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="up to 2\\^20 rows"): fp8_linear(torch.zeros(1, 256).expand((1 << 20) + 1, 256), w)
    with pytest.raises(RuntimeError, match="no CPU path"): rows.dequantize()


def test_logprobs_that_are_refused():
    x, t = torch.zeros(4, 100), torch.zeros(4, dtype=torch.int64)
    for bad in (x.double(), x[0], x[:, :0], torch.zeros(1).expand(4, 1 << 20), torch.zeros(1).expand((1 << 22) + 1, 8), torch.zeros(1).expand((1 << 21) + 1, 8193)):
        with pytest.raises(RuntimeError, match="token_logprobs expects logits"): token_logprobs(bad, t)
    for bad in (t.int(), t[:3], t[:, None], t.float()):
        with pytest.raises(RuntimeError, match="token_logprobs expects tokens"): token_logprobs(x, bad)
    for logits, top in ((x, -1), (x, 65), (x[:, :10], 11)):
        with pytest.raises(RuntimeError, match="alternatives"): token_logprobs(logits, t, top=top)
    with pytest.raises(RuntimeError, match="no CPU path"): token_logprobs(x, t, top=5)


CALLS = {
    "quantize": lambda t: quantize_fp8(t(X)), "norm x": lambda t: rms_norm_fp8(t(X), torch.ones(256)), "norm weight": lambda t: rms_norm_fp8(X, t(torch.ones(256))),
    "norm residual": lambda t: rms_norm_fp8(X, torch.ones(256), residual=t(X)), "weight": lambda t: FP8Weight(t(X)), "gated weight": lambda t: FP8Weight(X, t(X)),
    "linear": lambda t: fp8_linear(t(X), weight()), "gated": lambda t: fp8_gated(t(X), weight(gated=True)), "logprobs": lambda t: token_logprobs(t(X), torch.zeros(5, dtype=torch.int64)),
}


@pytest.mark.parametrize("name", CALLS)
def test_gradients_are_not_lost_without_a_word(name):
    need = lambda t: t.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"): CALLS[name](need)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"): CALLS[name](need)
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match="no backward pass"): CALLS[name](lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t)))


@pytest.mark.parametrize("name,args,message", [
    ("gaac_fp8_rows", [3, 16, 256, None, 0, None, 0.0, 5, 256, None, 16, 16, 16, 1, 0, None], "type must be"),
    ("gaac_fp8_rows", [0, 16, 256, None, 0, None, 0.0, 0, 256, None, 16, 16, 16, 1, 0, None], "bad sizes"),
    ("gaac_fp8_rows", [0, 16, 256, None, 0, None, 0.0, 5, 65537, None, 16, 16, 16, 1, 0, None], "bad sizes"),
    ("gaac_fp8_rows", [0, 16, 256, None, 0, 16, 0.0, 5, 32769, None, 16, 16, 16, 1, 0, None], "norm takes rows"),
    ("gaac_fp8_rows", [0, 16, 256, 16, 256, 16, 0.0, 5, 256, None, 16, 16, 16, 1, 0, None], "its sum together"),
    ("gaac_fp8_rows", [0, 16, 256, 16, 256, None, 0.0, 5, 256, 16, 16, 16, 16, 1, 0, None], "with the norm's weight"),
    ("gaac_fp8_rows", [0, 16, 256, None, 0, None, 0.0, 17, 256, None, 16, 16, 16, 1, 0, None], "bad sizes"),
    ("gaac_fp8_rows", [0, 16, 256, None, 0, None, 0.0, 5, 256, None, 16, 16, 16, 2, 0, None], "bad sizes"),
    ("gaac_fp8_rows", [0, 16, 256, None, 0, None, 0.0, 5, 256, None, 16, 16, 32, 2, 2, None], "bad sizes"),
    ("gaac_fp8_rows", [0, 16, 256, None, 0, None, 0.0, 5, 256, None, 24, 16, 16, 1, 0, None], "16-byte aligned"),
    ("gaac_fp8_values", [16, 16, 16, 1, 0, 17, 256, 16, 256, None], "bad sizes"),
    ("gaac_fp8_values", [24, 16, 16, 1, 0, 5, 256, 16, 256, None], "16-byte aligned"),
    ("gaac_fp8_product", [16, 16, 16, 16, 0, 64, 256, 0, 0, 16, 64, None], "bad sizes"),
    ("gaac_fp8_product", [16, 16, 16, 16, (1 << 20) + 1, 64, 256, 0, 0, 16, 64, None], "bad sizes"),
    ("gaac_fp8_product", [16, 16, 16, 16, 5, 64, 256, 0, 4, 16, 64, None], "type must be"),
    ("gaac_fp8_product", [16, 16, 24, 16, 5, 64, 256, 0, 0, 16, 64, None], "16-byte aligned"),
    ("gaac_logprobs", [0, 16, 100, 0, 100, 16, 0, None, 0, 16, 16, 16, None, None, None], "bad sizes"),
    ("gaac_logprobs", [0, 16, 100, (1 << 22) + 1, 100, 16, 0, None, 0, 16, 16, 16, None, None, None], "bad sizes"),
    ("gaac_logprobs", [0, 16, 8193, (1 << 21) + 1, 8193, 16, 0, 16, 1 << 40, 16, 16, 16, None, None, None], "bad sizes"),
    ("gaac_logprobs", [0, 16, 100, 4, 1 << 20, 16, 0, None, 0, 16, 16, 16, None, None, None], "bad sizes"),
    ("gaac_logprobs", [0, 16, 100, 4, 100, 16, 65, None, 0, 16, 16, 16, 16, 16, None], "alternatives"),
    ("gaac_logprobs", [0, 16, 100, 4, 100, 16, 5, None, 0, 16, 16, 16, None, 16, None], "alternatives"),
    ("gaac_logprobs", [0, 16, 9000, 4, 9000, 16, 5, 16, 4 * 2 * 56 - 1, 16, 16, 16, 16, 16, None], "work memory"),
    ("gaac_logprobs", [0, 17, 100, 4, 100, 16, 0, None, 0, 16, 16, 16, None, None, None], "not aligned"),
])
def test_the_library_refuses_before_it_launches(name, args, message):
    with pytest.raises(RuntimeError, match=f"{name} failed .*{message}"): _lib.call(name, *args)
