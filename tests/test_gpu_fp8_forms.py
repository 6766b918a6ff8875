"""Every form of the products of rows in 8 bits, with every end of K, on whole numbers whose sums are exact: an element that is lost, counted twice or scaled by another block's power is another result.

All partial sums are whole numbers below 2^24 (of one unit), which 32 bits hold in any order; elements are whole numbers of up to 3 bits times a power of two for each row and block, which 8 bits hold; and the products of eight
neighbours, at most 49 units of their own, lie within 2^6 of each other, so that nothing of them is cut.  Results are compared with equality, those of a gated block within silu's roundings."""
import pytest
import torch

from fp8_forms import CASES
from gaac_amd import FP8Weight, fp8_gated, fp8_linear, quantize_fp8
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
BF, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def gpu(): require_gpu()


def wholes(rows, K, seed, powers=3):
    """fp32 [rows, K]: +-1 .. +-7 times 1, 2 or 4 for each row and block of 128."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pick = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=g, device="cuda").float()
    scale = torch.exp2(pick(0, powers, rows, -(-K // 128))).repeat_interleave(128, 1)[:, :K]
    return pick(1, 8, rows, K) * (2 * pick(0, 2, rows, K) - 1) * scale


def sums(x, w):
    """x w^T in 64 bits, of which 32 bits hold every partial sum."""
    assert (x.abs().double() @ w.abs().double().T).max() < 1 << 24
    return x.double() @ w.double().T


def held(w):
    W = FP8Weight(w)
    assert torch.equal(W.dequantize().float(), w)
    return W


@pytest.mark.parametrize("form,M,N,K", [c[2:] for c in CASES if not c[0] and not c[1]])
def test_products(form, M, N, K):
    x, w = wholes(M, K, M + K), wholes(N, K, N + K)
    y, rows, W = sums(x, w).float(), quantize_fp8(x), held(w)
    for dtype in (BF, FP16): assert torch.equal(fp8_linear(rows, W, out_dtype=dtype), y.to(dtype))


@pytest.mark.parametrize("form,M,N,K", [c[2:] for c in CASES if c[0] and not c[1]])
def test_products_in_32_bits(form, M, N, K):
    x, w = wholes(M, K, M + K), wholes(N, K, N + K)
    assert torch.equal(fp8_linear(quantize_fp8(x), held(w), out_dtype=FP32), sums(x, w).float())


def check_gated(M, N, K, types):
    x, gate, up = wholes(M, K, M + K), wholes(N, K, N + K), wholes(N, K, N + K + 1)
    unit = 2.0 ** -10
    G = FP8Weight(gate * unit, up * unit)
    g, u = sums(x, gate) * unit, sums(x, up) * unit
    assert g.min() > -80
    y = g * torch.sigmoid(g) * u
    for dtype in types:
        f = torch.finfo(dtype)
        # silu: its exponential's argument is rounded to 24 bits (|g| 2^-23 of the result), then a few roundings of 2^-22; the product in 32 bits; the type's rounding
        tol = (2.0 ** -20 + g.abs() * 2.0 ** -22 + f.eps / 2 * 1.01) * y.abs() + f.smallest_normal * f.eps
        off = (fp8_gated(quantize_fp8(x), G, out_dtype=dtype).double() - y).abs()
        assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()}, by up to {(off / tol).max().item():.3g} of what is allowed"


@pytest.mark.parametrize("form,M,N,K", [c[2:] for c in CASES if not c[0] and c[1]])
def test_gated_blocks(form, M, N, K): check_gated(M, N, K, (BF, FP16))


@pytest.mark.parametrize("form,M,N,K", [c[2:] for c in CASES if c[0] and c[1]])
def test_gated_blocks_in_32_bits(form, M, N, K): check_gated(M, N, K, (FP32,))


@pytest.mark.parametrize("M,N,K", [(1, 20, 65536), (16, 40, 65531), (48, 64, 14336), (200, 300, 30000), (700, 900, 20000)])
def test_long_sums(M, N, K):
    """Every one of up to 65536 elements counts."""
    x, w = wholes(M, K, K), wholes(N, K, K + 1)
    y, rows, W = sums(x, w).float(), quantize_fp8(x), held(w)
    for dtype in (BF, FP16, FP32): assert torch.equal(fp8_linear(rows, W, out_dtype=dtype), y.to(dtype))


@pytest.mark.parametrize("wide,form,M,N,K", [(c[0], *c[2:]) for c in CASES if not c[1] and (c[0] or c[2] < 2) and c[5] > 500])
def test_exact_sums(wide, form, M, N, K):
    """Outputs in 32 bits, and those of 16 bits of up to 16 rows: in every block one element of both operands is 448, so that one product is 2^12 times its neighbours'.  The sum has all of these; the product of codes in 8 bits
    would cut them to multiples of 2^3."""
    x, w = wholes(M, K, M + K, powers=1), wholes(N, K, N + K, powers=1)
    blocks = -(-K // 128) // 2 * 2      # (an even number: what is large cancels)
    at = torch.arange(blocks, device="cuda") * 128 + torch.randint(0, 120, (blocks,), generator=torch.Generator().manual_seed(K)).cuda()
    x[:, at] = 448.0
    w[:, at] = 448.0 * (1 - 2.0 * (torch.arange(blocks, device="cuda") % 2))
    y = sums(x, w)
    near = (at // 8 * 8)[:, None] + torch.arange(8, device="cuda")      # neighbours of the large ones
    near = near[near != at[:, None]]
    lost = torch.stack([torch.fmod(row[near] * w[:, near], 8.0).double().sum(1) for row in x[:4]])
    for dtype in ((FP32,) if wide else (BF, FP16)):
        scale = 1.0 if wide else 2.0 ** -8
        want = (y * scale).float().to(dtype)
        assert ((y[:4] - lost) * scale).float().to(dtype).ne(want[:4]).float().mean() > 0.8      # (the test can tell)
        assert torch.equal(fp8_linear(quantize_fp8(x * scale), held(w), out_dtype=dtype), want)


@pytest.mark.parametrize("M", [1, 40])
def test_silu_far_below_zero(M):
    """Gates down to -80 by the formula; below -87, where 1 + e^-g leaves 32 bits, the result may be 0."""
    gates = torch.tensor([-0.5, -1, -8, -40, -72, -80, -88, -96, -104, -160, -448, 448, 80], device="cuda")
    G = FP8Weight(gates[:, None], torch.full((len(gates), 1), 2.0 ** 20, device="cuda"))
    out = fp8_gated(torch.ones(M, 1, device="cuda"), G, out_dtype=FP32).double()
    g = gates.double().expand(M, -1)
    y = g * torch.sigmoid(g) * 2.0 ** 20
    tol = (2.0 ** -20 + g.abs() * 2.0 ** -22) * y.abs() + torch.finfo(FP32).smallest_normal * 2.0 ** -23
    assert ((out - y).abs() <= torch.where(g < -87, y.abs() * 1.01, tol)).all()


def test_exact_sums_for_a_gated_block_in_bf16():
    """A result in 32 bits, rounded by the caller: what rounding the formula's value gives, but for elements next to a border.  Off by 2^-19 of itself (|g| up to 8; sums in 32 bits lose less for all but elements near 0),
    of borders 2^-8 apart, two sides: one element in 2^10, and as many again for what is near 0."""
    g = torch.Generator(device="cuda").manual_seed(3)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    M, N, K = 700, 2000, 1024
    x, G = quantize_fp8(normal(M, K)), FP8Weight(normal(N, K) * K ** -0.5, normal(N, K) * K ** -0.5)
    gate, up = (x.dequantize().double() @ w.double().T for w in G.dequantize())
    assert gate.abs().max() < 8
    want = (gate * torch.sigmoid(gate) * up).float().to(BF)
    assert fp8_gated(x, G, out_dtype=FP32).to(BF).ne(want).float().mean() < 2.0 ** -9
