"""Attention over the 4-bit cache against 64 bits with nothing allowed for but sums in 32 bits and the output's rounding, and over queries of every kind."""
import math

import pytest
import torch

import operators_ref as R
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
D = 128


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def attend(q, k, v, scale, nsplit=1):
    """One row over a cache that holds k, v; (output, k and v as held), on the CPU in 64 bits."""
    from gaac_amd import FP4KVCache
    c = FP4KVCache(1, k.shape[1], k.shape[0])
    c.prefill(0, k.cuda(), v.cuda())
    out = c.attention(q[None].cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"), scale, nsplit=nsplit)
    return out[0].double().cpu(), R.stored(k), R.stored(v)


def bound(q, k, v, scale):
    """(definition, largest error), fp64 [n_q, 128].

    A score: 128 products summed in 32 bits (128 * 2^-24 of the sum of their magnitudes), and what the query's two operands leave out, at most 2^-21 of the head's largest
    element on each channel below 2^-13 of it; times scale and minus the maximum, two roundings more of 2^-24 of the largest score; each counts twice, in the weight and in the sum.  exp2 is off
    by 2^-22, a weight's two parts of 8 bits leave out 2^-16 of it, the sums over the tokens are off by 2^-24 a token, and the output is rounded to bf16: half a step, 2^-8 of
    itself."""
    q = q.double()
    n_q, n_kv = q.shape[0], k.shape[1]
    G = n_q // n_kv
    out, tol = torch.zeros(n_q, D, dtype=torch.float64), torch.zeros(n_q, D, dtype=torch.float64)
    for h in range(n_kv):
        qh, kh, vh = q[h * G:(h + 1) * G], k[:, h], v[:, h]
        p = torch.softmax(qh @ kh.T * scale, -1)
        size = (qh.abs() @ kh.abs().T * abs(scale)).amax(-1, keepdim=True)
        top = qh.abs().amax(-1, keepdim=True)
        left = (2.0 ** -21 * top * (qh.abs() < 2.0 ** -13 * top) @ kh.abs().T * abs(scale)).amax(-1, keepdim=True)
        out[h * G:(h + 1) * G] = p @ vh
        rel = 2 * (130 * 2.0 ** -24 * size + left) + 2.0 ** -20 + 2.0 ** -16 + len(kh) * 2.0 ** -24
        tol[h * G:(h + 1) * G] = rel * (p @ vh.abs()) * 1.01 + 2.0 ** -8 * out[h * G:(h + 1) * G].abs() + 1e-37
    return out, tol


def check(q, k, v, scale, nsplit=1):
    out, hk, hv = attend(q, k, v, scale, nsplit)
    ref, tol = bound(q, hk, hv, scale)
    err = (out - ref).abs()
    assert (err <= tol).all(), f"{(err / tol).max():.3g} of the bound"


@pytest.mark.parametrize("L,nsplit", [(2, 1), (3, 1), (17, 1), (64, 1), (64, 2), (300, 1), (300, 5), (3000, 1), (3000, 8)])
@pytest.mark.parametrize("n_kv,G", [(8, 4), (1, 16), (3, 1)])
def test_weights_keep_their_bits_where_values_cancel(L, nsplit, n_kv, G):
    """Every second token's values are the negative of the one before: what is left of the sum is far smaller than its terms, so a weight's rounding to 8 bits would
    show."""
    require_gpu()
    k, v, q = rnd(L, n_kv, D, seed=1), rnd(L, n_kv, D, seed=2), rnd(n_kv * G, D, seed=3)
    v[1::2] = -v[0::2][:len(v[1::2])]
    check(q, k, v, D ** -0.5, nsplit)
    check(q, k / 16, v, D ** -0.5, nsplit)


@pytest.mark.parametrize("up", [2.0 ** 6, 2.0 ** 12, 2.0 ** 15, 2.0 ** 24])
@pytest.mark.parametrize("where", [[5], [0, 64, 127], [77, 78]])
def test_queries_with_channels_far_above_the_others(up, where):
    """Channels of a query 64 to 2^24 times as large as the rest, over keys that have little or nothing there, so that the rest decides."""
    require_gpu()
    n_kv, G, L = 2, 4, 200
    q, k, v = rnd(n_kv * G, D, seed=1), rnd(L, n_kv, D, seed=2), rnd(L, n_kv, D, seed=3)
    q[:, where] *= up
    for small in (0.0, 1.0 / up):
        kk = k.clone()
        kk[:, :, where] *= small
        check(q, kk, v, D ** -0.5)


@pytest.mark.parametrize("size", [0.0, 2.0 ** -133, 2.0 ** -126, 2.0 ** -100, 2.0 ** 60])
def test_queries_of_every_size(size):
    """Zeros, the smallest numbers (subnormal ones among them) and large ones; keys and scale take the scores back into range."""
    require_gpu()
    n_kv, G, L = 2, 4, 100
    q = (rnd(n_kv * G, D, seed=1).double() * size).to(torch.bfloat16)
    k, v = rnd(L, n_kv, D, seed=2), rnd(L, n_kv, D, seed=3)
    check(q, k, v, 1.0 if size <= 1 else D ** -0.5 / size)
    if 0 < size < 1: check(q, (k.double() * 2.0 ** 100).to(torch.bfloat16), v, min(D ** -0.5 / (size * 2.0 ** 100), 2.0 ** 30))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("nsplit", [1, 3])
def test_a_query_that_is_not_finite_is_nan_and_the_others_are_as_without_it(bad, nsplit):
    require_gpu()
    n_kv, G, L = 2, 5, 150
    q, k, v = rnd(n_kv * G, D, seed=1), rnd(L, n_kv, D, seed=2), rnd(L, n_kv, D, seed=3)
    clean, _, _ = attend(q, k, v, D ** -0.5, nsplit)
    for head, ch in ((0, 0), (3, 127), (7, 64), (9, 31)):
        x = q.clone()
        x[head, ch] = bad
        out, _, _ = attend(x, k, v, D ** -0.5, nsplit)
        others = torch.arange(n_kv * G) != head
        assert out[head].isnan().all() and torch.equal(out[others], clean[others])
