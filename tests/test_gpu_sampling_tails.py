"""Sampling where many small weights make up the sum, against the stated bound: a weight is off by at most 2^-44 of the largest, a sum by that for each of its tokens."""
import numpy as np
import pytest
import torch

from gaac_amd import sample
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu


def within_the_bound(x, u, token, kept=None):
    """Whether `token` may come: u * total lies in its stretch of the running sum, both taken to 64 bits of mantissa, give or take n * 2^-44 for each of the three sums
    and 2^-52 of the total for the shares."""
    kept = np.arange(len(x)) if kept is None else np.sort(kept)
    x = x.astype(np.longdouble)
    w = np.exp(x - x.max())[kept]
    run = np.cumsum(w)
    tol = 2 * len(kept) * 2.0 ** -44 + run[-1] * 2.0 ** -52
    at = int(np.searchsorted(kept, token))
    assert kept[at] == token and w[at] >= 2.0 ** -44 * (1 - 2.0 ** -40)
    want = np.longdouble(u) * run[-1]
    return (run[at - 1] if at else 0) - tol <= want <= run[at] + tol


TOP_U = 1 - 2.0 ** -24
TAILS = [(1048560, -30.3), (1048560, -29.0), (1048560, -20.0), (128256, -30.4), (128256, -27.5), (128256, -12.0), (4000, -30.0)]


@pytest.mark.parametrize("V,tail", TAILS)
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_long_flat_tails(V, tail, at):
    """One token far above all others, which are alike: with u next to 1 the draw falls among them."""
    require_gpu()
    x = torch.full((V,), tail)
    x[dict(first=0, middle=V // 2, last=V - 1)[at]] = 0
    us = [0.0, 0.5, 1 - 2.0 ** -20, 1 - 2.0 ** -23, TOP_U]
    got = sample(x.cuda().expand(len(us), -1), torch.tensor(us, dtype=torch.float32, device="cuda"))
    for u, t in zip(us, got.tolist()): assert within_the_bound(x.numpy(), u, t), f"u {u}: {t}"


@pytest.mark.parametrize("V", [1048560, 128256, 4000])
def test_a_tail_below_the_resolution_never_comes(V):
    require_gpu()
    x = torch.full((3, V), -31.0)
    x[:, V // 3] = 0
    for settings in ({}, dict(top_p=0.999999), dict(top_k=V // 2), dict(min_p=1e-30)):
        assert sample(x.cuda(), torch.tensor([0.0, 0.5, TOP_U], device="cuda"), **settings).tolist() == [V // 3] * 3


@pytest.mark.parametrize("V", [1048560, 128256])
@pytest.mark.parametrize("top_k", [0, 70000])
def test_tails_of_many_sizes(V, top_k):
    """Weights over the whole range down to the resolution, drawn along the whole sum, with and without a prefix of the order."""
    require_gpu()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(V, generator=g) * 6 - 12
    x[1000], x[V - 7] = 1.5, 4.0
    us = torch.cat([torch.rand(20, generator=g), 1 - torch.exp2(-torch.arange(1.0, 25))])
    got = sample(x.cuda().expand(len(us), -1), us.cuda(), top_k=top_k)
    kept = np.lexsort((np.arange(V), -x.numpy()))[:top_k] if top_k else None
    for u, t in zip(us.tolist(), got.tolist()): assert within_the_bound(x.numpy(), u, t, kept), f"u {u}: {t}"


@pytest.mark.parametrize("tail", [-30.3, -28.0, -16.0])
def test_a_share_of_a_long_tail(tail):
    """top_p close to 1: as many of the equals are kept as make up the share, give or take what the bound allows."""
    require_gpu()
    V, p = 1048560, 1 - 2.0 ** -24
    x = torch.full((V,), tail)
    x[5] = 0
    w = float(np.exp(np.longdouble(tail)))
    t = int(sample(x.cuda()[None], torch.tensor([TOP_U], device="cuda"), top_p=p))
    total, tol = 1 + (V - 1) * w, V * 2.0 ** -44 + 2.0 ** -52 * V
    most = (p * total + tol - 1) / max(w - 2.0 ** -44, 2.0 ** -44) + 2      # tokens of the tail that may be kept
    assert t == 5 or 0 <= t <= min(most, V)
