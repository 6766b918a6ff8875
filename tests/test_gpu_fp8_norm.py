"""The norm before rows in 8 bits, code by code: results below and beyond what 32 bits hold, results next to a border between two codes.

The kernel has y in 64 bits, off by a few 2^-52 of itself, so its codes are the formula's wherever y is not that near to a border; rows here are equal to the definition, without a tolerance."""
import pytest
import torch

import fp8_ref as R
from gaac_amd import FP8Weight, _lib, fp8_linear, rms_norm_fp8
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True, params=["binding", "ctypes"])
def gpu(request, monkeypatch):
    require_gpu()
    if request.param == "ctypes": monkeypatch.setattr(_lib, "_calls", _lib._CtypesCalls())


def rnd(*shape, seed=0, dtype=BF):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def codes_of(x, w, eps, residual=None):
    """rms_norm_fp8's values, fp64 on the CPU, and those of the definition: of the sum in 32 bits, where there is a residual."""
    dev = lambda t: None if t is None else t.cuda()
    out = rms_norm_fp8(dev(x), dev(w), eps, residual=dev(residual))
    return (out if residual is None else out[0]).dequantize().double().cpu(), R.stored(R.norm(x if residual is None else x.float() + residual.float(), w, eps)[0])


def same(a, b):
    assert torch.equal(a.isnan(), b.isnan()), f"{int(a.isnan().sum())} NaN, {int(b.isnan().sum())} by the definition"
    assert torch.equal(a.nan_to_num(0), b.nan_to_num(0)), f"{int((a != b).sum())} of {a.numel()} codes differ"


@pytest.mark.parametrize("dtype", [BF, FP32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K", [(1, 128), (3, 300), (17, 4096), (5, 5000), (2, 20000)])
def test_results_that_32_bits_round_to_zero(M, K, residual, dtype):
    """Elements of ordinary rows with h * weight from 1e-44 to 1e-60, of both signs: 0 in 8 bits, and what is beside them by the definition."""
    x, w = rnd(M, K, seed=K, dtype=dtype), torch.rand(K, generator=torch.Generator().manual_seed(1)).to(dtype) + 0.5
    r = rnd(M, K, seed=K + 1, dtype=dtype) if residual else None
    at = torch.arange(5, K, 37)
    w[at] = (10.0 ** -torch.linspace(24, 30, len(at)).double()).to(dtype)
    x[:, at] = ((10.0 ** -torch.linspace(20, 30, len(at)).double()) * torch.where(torch.arange(len(at)) % 3 == 0, -1, 1)).to(dtype)
    if residual: r[:, at] = 0
    w[at[-1]] = -w[at[-1]]
    got, want = codes_of(x, w, 1e-5, r)
    same(got, want)
    assert (got[:, at] == 0).all()
    out = fp8_linear(rms_norm_fp8(x.cuda(), w.cuda(), 1e-5), FP8Weight(rnd(20, K, seed=3).cuda()))
    assert out.isfinite().all()
    # blocks with nothing else, in rows that have other blocks
    if K > 128:
        w[:128], x[:, :128] = 1e-25, 1e-25
        if residual: r[:, :128] = 0
        got, want = codes_of(x, w, 1e-5, r)
        same(got, want)
        assert (got[:, :128] == 0).all() and (got[:, 128:] != 0).any()


def test_one_element_far_above_another():
    for dtype in (BF, FP32):
        x = torch.zeros(1, 128, dtype=dtype)
        x[0, 3], x[0, 70] = 1e20, 1e-27
        got, want = codes_of(x, torch.ones(128, dtype=dtype), 1e-6)
        same(got, want)
        assert got[0, 70] == 0 and got[0, 3] == 11      # sqrt(128) is 11.3


@pytest.mark.parametrize("dtype", [BF, FP32])
def test_results_beyond_32_bits(dtype):
    """A finite result beyond the largest number of 32 bits is held as 448 * 2^119, as every result beyond that is."""
    x, w = rnd(6, 700, seed=4, dtype=dtype), torch.full((700,), 2.9e38, dtype=dtype)
    w[300:] = 3.0
    got, want = codes_of(x, w, 1e-5)
    same(got, want)
    assert got.isfinite().all() and got.abs().max() == 448 * 2.0 ** 119 and (got[:, :256].abs() == got.abs().max()).any(1).all()
    x[2, 5], w[310] = torch.inf, torch.inf      # what is not finite stays so
    got, want = codes_of(x, w, 1e-5)
    assert got[[0, 1, 3, 4, 5], 256:384].isnan().all() and got[[0, 1, 3, 4, 5], :256].isfinite().all() and got[2, :128].isnan().all() and (got[2, 128:256] == 0).all()


@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K", [(1, 1), (4, 4096), (17, 129), (5, 5000), (700, 512), (3, 32768), (130, 14336), (2500, 1024)])
def test_codes_are_the_formulas(M, K, residual, dtype):
    x, w, r = rnd(M, K, seed=1, dtype=dtype), rnd(K, seed=2, dtype=dtype), rnd(M, K, seed=3, dtype=dtype) if residual else None
    same(*codes_of(x, w, 1e-5, r))


def next_to_borders(x, eps, seed):
    """A weight fp32 [K] for a row x fp32 [1, K] with which every y lies next to a border between two codes, nearer than half a step of 32 bits: targets are the middles of the grid's values from 2^-6 to 448
    in blocks whose largest element is 440, and in every third block 448 itself, the border between two powers of two."""
    K = x.shape[1]
    g = torch.Generator().manual_seed(seed)
    middles = ((R.GRID[1:] + R.GRID[:-1]) / 2)[8:]
    target = middles[torch.randint(0, len(middles), (K,), generator=g)]
    target[::128] = 440.0
    target[::384] = 448.0
    h = x.double()
    r = 1 / torch.sqrt((h * h).mean() + eps)
    w = (target / (h[0] * r)).float()
    off = (h[0] * r * w.double() - target) / target
    assert (off.abs() > 2.0 ** -45).all() and (off.abs() < 2.0 ** -23).all()
    return w


@pytest.mark.parametrize("scale,eps", [(1.0, 1e-5), (1e-4, 0.1), (0.02, 1e-3), (1e-20, 1e-6)])
@pytest.mark.parametrize("seed", range(3))
def test_results_next_to_a_border(seed, scale, eps):
    """What a norm in 32 bits, or one rounded to 32 bits before it is rounded to 8, would get wrong.  eps is a number of 32 bits."""
    eps = torch.tensor(eps).double().item()
    x = (torch.rand(1, 3000, generator=torch.Generator().manual_seed(seed)) + 0.5) * scale
    w = next_to_borders(x, eps, seed + 10)
    y, _ = R.norm(x, w, eps)
    want = R.stored(y)
    twice = R.stored(y.float())
    assert (want != twice).sum() > 3000 / 8      # (the test can tell: rounded twice, these are other codes)
    same(codes_of(x, w, eps)[0], want)
    same(codes_of(x, w, eps, torch.zeros_like(x))[0], want)
