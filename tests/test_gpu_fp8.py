"""Rows and weights in 8 bits, the norm before them, products and gated blocks, against their definitions in 64 bits."""
import pytest
import torch

import fp8_ref as R
from gaac_amd import FP8Rows, FP8Weight, fp8_gated, fp8_linear, quantize_fp8, rms_norm_fp8
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def gpu(): require_gpu()


def rnd(*shape, seed=0, dtype=BF, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * torch.exp2(torch.rand(shape[-1], generator=g) * 2 * spread - spread)).to(dtype).cuda()


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    assert a.shape == b.shape and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0), b.nan_to_num(0))


def within(a, y, tol):
    a = a.double().cpu()
    assert a.shape == y.shape and torch.equal(a.isnan(), y.isnan())
    off = (a - y).abs().nan_to_num(0) - tol.nan_to_num(0)
    assert (off <= 0).all(), f"{int((off > 0).sum())} of {off.numel()} too far off, by up to {off.max().item():.3g}"


# ---------------------------------------------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (16, 129), (17, 640), (5, 5000), (33, 4096), (300, 1000), (2, 14336), (1, 65536), (1500, 264)])
def test_rows_hold_their_definition(M, K, dtype):
    x = rnd(M, K, seed=M + K, dtype=dtype)
    r = quantize_fp8(x)
    assert r.shape == (M, K) and r.nbytes <= -(-M // 16) * 16 * (-(-K // 128) * 128 + 4 * -(-K // 512))
    same(r.dequantize(), R.stored(x))


def test_every_value_and_tie_of_the_grid():
    grid = torch.cat([R.GRID, (R.GRID[1:] + R.GRID[:-1]) / 2, (R.GRID[1:] * 0.99 + R.GRID[:-1] * 0.01)])
    grid = torch.cat([grid, -grid])
    rows = []
    for i in range(0, len(grid), 126):      # with 448 in each block the power is 2^0
        part = grid[i:i + 126]
        rows.append(torch.cat([torch.tensor([448.0, -448.0], dtype=torch.float64), part, torch.zeros(126 - len(part), dtype=torch.float64)]))
    x = torch.stack(rows)
    for power in (-100, -20, 0, 7, 100):
        y = (x * 2.0 ** power).float()
        same(quantize_fp8(y.cuda()).dequantize(), R.stored(y))


def test_blocks_at_the_ends_of_the_range():
    x = torch.zeros(20, 256)
    tiny, huge = 2.0 ** -149, torch.finfo(FP32).max
    for i, v in enumerate([0.0, tiny, 2.0 ** -126, 2.0 ** -120, 448 * 2.0 ** -117, 449 * 2.0 ** -117, 448.0, 448.0001, 464.0, 480.0, 512.0, huge, 448 * 2.0 ** 119]): x[i, 5], x[i, 200] = v, -v / 2
    x[13, 3], x[14, 3], x[15, 3], x[16, 130] = torch.inf, -torch.inf, torch.nan, torch.nan
    x[13, 7] = 1
    v = quantize_fp8(x.cuda()).dequantize()
    same(v, R.stored(x))
    assert v[13, :128].isnan().all() and (v[13, 128:] == 0).all() and v[16, 128:].isnan().all()


@pytest.mark.parametrize("dtype", [BF, FP32])
def test_rows_of_other_strides(dtype):
    wide = rnd(40, 1030, seed=3, dtype=dtype)
    for x in (wide[:, :1024], wide[:, 3:900], wide[::2, 8:520], wide.t()[:64], wide[:1].expand(20, 1030), wide[:, :1], wide.flip(0)):
        same(quantize_fp8(x).dequantize(), R.stored(x))
    assert quantize_fp8(wide[:0]).dequantize().shape == (0, 1030)


@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K", [(1, 1), (4, 4096), (17, 129), (5, 5000), (700, 512), (3, 32768), (130, 14336), (2500, 1024)])
def test_norm(M, K, residual, dtype):
    x, w, r = rnd(M, K, seed=1, dtype=dtype), rnd(K, seed=2, dtype=dtype, spread=0.5), rnd(M, K, seed=3, dtype=dtype) if residual else None
    y, h = R.norm(x, w, 1e-5, r)
    out = rms_norm_fp8(x, w, 1e-5, residual=r)
    if residual:
        out, got = out
        assert got.dtype == dtype and got.is_contiguous()
        within(got, h, torch.finfo(dtype).eps / 2 * h.abs() * 1.01 + 1e-7)
    within(out.dequantize(), y, R.half_step(y) * (1 + 2.0 ** -20) + y.abs() * 2.0 ** -22)      # (nearest values; y in 64 bits, rounded to 32)


def test_norm_of_special_rows():
    x = rnd(6, 300, seed=4, dtype=FP32)
    x[1] = 0
    x[2, 5], x[3, 7] = torch.inf, torch.nan
    x[4] *= 1e30
    w = torch.ones(300, device="cuda")
    v = rms_norm_fp8(x, w, 1e-6).dequantize()
    assert (v[1] == 0).all() and v[2, :128].isnan().all() and (v[2, 128:] == 0).all() and v[3].isnan().all()
    y, _ = R.norm(x[4:], w, 1e-6)
    within(v[4:], y, R.half_step(y) * 1.001)
    wide = rnd(40, 1030, seed=5)
    for x in (wide[:, 3:900], wide[::2, 8:520], wide.t()[:64]):      # strides
        w = rnd(x.shape[1], seed=6)
        got, h = rms_norm_fp8(x, w, residual=x)
        same(got.dequantize(), rms_norm_fp8(x.contiguous(), w, residual=x.contiguous())[0].dequantize())
        same(h, (x.float() + x.float()).to(BF))
        same(rms_norm_fp8(x, rnd(2 * x.shape[1], seed=6)[::2]).dequantize(), rms_norm_fp8(x, rnd(2 * x.shape[1], seed=6)[::2].clone()).dequantize())


# ---------------------------------------------------------------------------------------------------- products
SHAPES = [(1, 1, 1), (1, 16, 128), (2, 17, 129), (15, 100, 640), (16, 1000, 512), (17, 33, 1000), (33, 48, 384), (64, 256, 256), (65, 130, 2000), (130, 513, 300), (257, 300, 1100), (600, 260, 512),
          (4, 4096, 4096), (48, 64, 14336), (1, 20, 65536), (1000, 1000, 256), (520, 2050, 128)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
def test_products(M, N, K, dtype):
    x, w = rnd(M, K, seed=M + N, dtype=dtype), rnd(N, K, seed=K, dtype=dtype, spread=1.0)
    W = FP8Weight(w)
    assert (W.N, W.K, W.gated) == (N, K, False)
    same(W.dequantize(), R.stored(w))
    out = fp8_linear(x, W)
    assert out.dtype == dtype
    within(out, *R.product(R.stored(x), R.stored(w), dtype))
    rows = quantize_fp8(x)
    for t in (BF, FP16, FP32): assert torch.equal(fp8_linear(rows, W, out_dtype=t), fp8_linear(x, W, out_dtype=t))
    assert fp8_linear(rows, W).dtype == BF


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [BF, FP32])
def test_gated_blocks(M, N, K, dtype):
    x, a, b = rnd(M, K, seed=M + N, dtype=dtype), rnd(N, K, seed=K), rnd(N, K, seed=K + 1)
    a, b = a * K ** -0.5, b * K ** -0.5
    W = FP8Weight(a, b)
    assert (W.N, W.K, W.gated) == (N, K, True)
    for v, t in zip(W.dequantize(), (a, b)): same(v, R.stored(t))
    for t in (BF, FP16, FP32): within(fp8_gated(x, W, out_dtype=t), *R.gated(R.stored(x), R.stored(a), R.stored(b), t))
    out = fp8_gated(x, W)
    assert out.dtype == BF
    rows = fp8_gated(x, W, quantize=True)
    assert isinstance(rows, FP8Rows) and rows.shape == (M, N)
    same(rows.dequantize(), R.stored(out))


# sizes at which the forms that the smaller ones do not reach are taken: blocks of 4 x 2 tiles, of 64 x 128, 128 x 128 and 256 x 256 outputs; each with rows, columns and inputs that end inside a tile, and exponents inside a dword
@pytest.mark.parametrize("M,N,K", [(150, 2000, 2100), (40, 9000, 1100), (300, 4100, 1300), (1100, 3700, 900), (700, 4100, 1000), (3000, 2100, 129), (4097, 5000, 650), (4111, 4999, 140), (3300, 4200, 200)])
@pytest.mark.parametrize("dtype", [BF, FP16, FP32])
def test_larger_products(M, N, K, dtype):
    x, a, b = rnd(M, K, seed=M, dtype=dtype), rnd(N, K, seed=N), rnd(N, K, seed=N + 1)
    a, b = a * K ** -0.5, b * K ** -0.5
    X = R.stored(x)
    within(fp8_linear(x, FP8Weight(a)), *R.product(X, R.stored(a), dtype))
    within(fp8_gated(x, FP8Weight(a, b), out_dtype=dtype), *R.gated(X, R.stored(a), R.stored(b), dtype))


# blocks of 192 x 128 outputs go through K in turns of twelve blocks, and every number of blocks that is left has an end of its own
@pytest.mark.parametrize("blocks", [2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 19, 24])
def test_every_end_of_the_inputs(blocks):
    M, N, K = 770, 6100, 128 * blocks - 5
    x, a = rnd(M, K, seed=blocks), rnd(N, K, seed=blocks + 1) * K ** -0.5
    X, A = R.stored(x), R.stored(a)
    within(fp8_linear(x, FP8Weight(a)), *R.product(X, A, BF))
    gate, up = a[:3050], a[3050:]
    within(fp8_gated(x, FP8Weight(gate, up)), *R.gated(X, R.stored(gate), R.stored(up), BF))


@pytest.mark.parametrize("M", [1, 16, 40, 300, 700])
def test_a_row_that_is_not_finite_is_its_own_matter(M):
    x, w = rnd(M, 700, seed=8), rnd(600, 700, seed=9)
    clean = fp8_linear(x, FP8Weight(w))
    x[M // 2, 650] = torch.nan
    w[33, 0], w[599, 699] = torch.inf, torch.nan
    out = fp8_linear(x, FP8Weight(w))
    bad = torch.zeros(M, 600, dtype=torch.bool, device="cuda")
    bad[M // 2], bad[:, 33], bad[:, 599] = True, True, True
    assert out[bad].isnan().all() and torch.equal(out[~bad], clean[~bad])
    empty = fp8_linear(x[:0], FP8Weight(w))
    assert empty.shape == (0, 600) and fp8_gated(x[:0], FP8Weight(w, w)).shape == (0, 600) and fp8_gated(x[:0], FP8Weight(w, w), quantize=True).shape == (0, 600)


def test_values_far_apart_and_far_out():
    """Exponents of both operands at both ends; the sum's order of size is theirs."""
    for px, pw in ((110, -110), (-100, 60), (40, 60), (0, 0)):
        x, w = rnd(20, 384, seed=11, dtype=FP32, spread=8.0) * 2.0 ** px, rnd(40, 384, seed=12, dtype=FP32, spread=8.0) * 2.0 ** pw
        within(fp8_linear(x, FP8Weight(w)), *R.product(R.stored(x), R.stored(w), FP32))
