"""Sampling on the GPU against its definition in 64 bits: the same token, always."""
import math

import numpy as np
import pytest
import torch

import operators_ref as R
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50, top_p=0.95), dict(top_p=0.9), dict(top_p=0.5, min_p=0.02), dict(min_p=0.1), dict(top_k=1), dict(top_k=7, temperature=2.0),
            dict(temperature=0.2, top_p=0.999), dict(temperature=1.5, top_k=1000, min_p=0.001), dict(top_p=0.0), dict(top_p=1e-9, top_k=3), dict(temperature=1e-3, top_k=20), dict(temperature=1e30, top_p=0.7),
            dict(temperature=1e-30, top_k=5), dict(min_p=1.0), dict(min_p=5.0, top_k=9), dict(temperature=math.inf, top_k=11), dict(temperature=100.0, top_p=0.3, top_k=400)]


def logits(B, V, dtype, seed=0, kind="model"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * 2.5
    if kind == "model":
        x.scatter_add_(1, torch.randint(0, V, (B, 20), generator=g), torch.rand(B, 20, generator=g) * 10)
        x[torch.rand(B, V, generator=g) < 0.1] = -math.inf
    elif kind == "flat": x = x * 0.01
    elif kind == "equal": x = torch.full((B, V), 1.25)
    elif kind == "few values": x = torch.round(x)
    elif kind == "zeros of both signs": x = torch.where(x > 0, 0.0, -0.0)
    elif kind == "wide": x = x * 1000
    elif kind == "lowest": x = torch.where(torch.rand(B, V, generator=g) < 0.9, torch.finfo(dtype).min, x)
    return x.to(dtype), torch.rand(B, generator=g)


def check(x, u, got, **settings):
    B = x.shape[0]
    row = lambda name, default: [float(v) for v in settings[name].cpu()] if isinstance(settings.get(name), torch.Tensor) else [float(np.float32(settings.get(name, default)))] * B
    t, k, p, m = row("temperature", 1.0), row("top_k", 0), row("top_p", 1.0), row("min_p", 0.0)
    want = [R.sample(x[b].double().cpu().numpy(), float(u[b]), t[b], int(k[b]), p[b], m[b]) for b in range(B)]
    assert got.dtype == torch.int64 and got.tolist() == want


@pytest.mark.parametrize("kind", ["model", "flat", "equal", "few values", "zeros of both signs", "wide", "lowest"])
@pytest.mark.parametrize("dtype", TYPES)
def test_settings(dtype, kind):
    from gaac_amd import sample
    require_gpu()
    for i, s in enumerate(SETTINGS):
        x, u = logits(4, 5003, dtype, i, kind)
        check(x, u, sample(x.cuda(), u.cuda(), **s), **s)


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 511, 512, 513, 1000, 4096, 32000, 50257, 128256, 151936, 262144, 1048560])
@pytest.mark.parametrize("dtype", TYPES)
def test_vocabularies(dtype, V):
    """Odd sizes leave rows at every alignment."""
    from gaac_amd import sample
    require_gpu()
    for i, s in enumerate((dict(temperature=0.7, top_k=50, top_p=0.95), dict(top_p=0.9, min_p=0.001), dict(temperature=0.0), dict(top_k=V - 1) if V > 1 else dict())):
        x, u = logits(3, V, dtype, i)
        if V < 10: x = torch.where(torch.isinf(x), 0.5, x)
        check(x, u, sample(x.cuda(), u.cuda(), **s), **s)


def test_settings_for_each_row():
    from gaac_amd import sample
    require_gpu()
    B = 40
    x, u = logits(B, 3001, torch.float32)
    i = torch.arange(B)
    s = dict(temperature=torch.where(i % 5 == 0, 0.0, 0.3 + 0.1 * (i % 9)), top_k=torch.where(i % 3 == 0, 30, -1 + i % 2).int(), top_p=torch.where(i % 4 == 1, 1.0, 0.9), min_p=torch.where(i % 2 == 1, 0.0, 0.05))
    check(x, u, sample(x.cuda(), u.cuda(), **{k: v.cuda() for k, v in s.items()}), **s)


def test_random_numbers_at_the_ends_and_beyond():
    from gaac_amd import sample
    require_gpu()
    us = [0.0, 1 - 2.0 ** -24, 1.0, 7.0, -0.5, math.nan, math.inf, 2.0 ** -149]
    x = logits(1, 1000, torch.bfloat16)[0].repeat(len(us), 1)
    u = torch.tensor(us)
    for s in (dict(), dict(top_k=10), dict(top_p=0.5)): check(x, u, sample(x.cuda(), u.cuda(), **s), **s)


def test_rows_that_have_little_to_choose_from():
    from gaac_amd import sample
    require_gpu()
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf] * 6, [nan] * 6, [-inf, nan, -inf, nan, 3.0, -inf], [nan, 1.0, nan, 2.0, nan, nan], [inf, 1.0, inf, 2.0, nan, inf], [-inf, 0.0, -inf, 0.0, -inf, 0.0]])
    for dtype in TYPES:
        for s in (dict(), dict(temperature=0.0), dict(top_k=2), dict(top_p=0.5), dict(top_k=4, top_p=0.9, min_p=0.1)):
            for u0 in (0.0, 0.4, 0.99):
                u = torch.full((6,), u0)
                got = sample(x.to(dtype).cuda(), u.cuda(), **s)
                assert got[:2].tolist() == [-1, -1] and got[2] == 4
                check(x.to(dtype), u, got, **s)


def test_every_boundary_of_a_distribution():
    """u just below, at and above each running sum of equal weights: the first token whose sum exceeds u times the total."""
    from gaac_amd import sample
    require_gpu()
    V = 64
    x = torch.zeros(3 * V, V)
    u = torch.cat([torch.arange(V) / V, torch.nextafter(torch.arange(1, V + 1) / V, torch.tensor(0.0)), torch.nextafter(torch.arange(V) / V, torch.tensor(1.0))])
    got = sample(x.cuda(), u.cuda())
    assert got.tolist() == list(range(V)) * 3
    # half of them by top_p: the lower half of the indices
    got = sample(x.cuda(), u.cuda(), top_p=0.5)
    assert got.tolist() == [int(v * 32) for v in u.tolist()]


def test_shares_of_a_distribution():
    """Over evenly spaced u each token comes as often as its weight says, to within one."""
    from gaac_amd import sample
    require_gpu()
    n, V = 4096, 33
    x = (torch.randn(V, generator=torch.Generator().manual_seed(1)) * 1.5).to(torch.bfloat16)
    u = (torch.arange(n) + 0.5) / n
    got = torch.bincount(sample(x.repeat(n, 1).cuda(), u.cuda(), temperature=0.8).cpu(), minlength=V)
    p = torch.softmax(x.double() / float(np.float32(0.8)), 0)
    assert ((got - n * p).abs() <= 1.0).all()


def test_layouts_and_graphs():
    from gaac_amd import sample
    require_gpu()
    x, u = logits(6, 2 * 777, torch.bfloat16)
    x, u = x.cuda(), u.cuda()
    s = dict(temperature=0.9, top_k=40, top_p=0.9)
    for view in (x[:, 5:705], x[::2, 3:], x[:, ::2], x[:1].expand(6, -1), x[:0]):
        uu = u[:view.shape[0]]
        check(view.cpu(), uu, sample(view, uu, **s), **s)
    both = torch.stack([u, u], 1)[:, 0]
    check(x.cpu(), u, sample(x, both, **s), **s)
    buf, ub = x.clone(), u.clone()
    sample(buf, ub, **s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g): got = sample(buf, ub, **s)
    for step in range(4):
        buf.copy_(x.roll(step, 0)); ub.copy_(u.roll(step * 2, 0))
        g.replay()
        torch.cuda.synchronize()
        check(buf.cpu(), ub, got, **s)


def test_many_rows():
    from gaac_amd import sample
    require_gpu()
    x, u = logits(700, 900, torch.float16)
    s = dict(temperature=1.1, top_p=0.8)
    check(x, u, sample(x.cuda(), u.cuda(), **s), **s)


@pytest.mark.parametrize("B,V", [(70000, 5), (1025, 4090), (2300, 4200)])
def test_more_rows_than_a_launch_takes(B, V):
    """Settings, random numbers and tokens of the rows behind the first launches' are their own; a few rows are drawn by the definition, and all rows alike in one call and in pieces."""
    from gaac_amd import sample
    require_gpu()
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randn(B, V, generator=g, device="cuda") * 3).to(torch.bfloat16)
    u = torch.rand(B, generator=g, device="cuda")
    i = torch.arange(B, device="cuda")
    s = dict(temperature=torch.where(i % 3 == 0, 0.0, 0.5 + (i % 5) * 0.3), top_k=(i % 7).int(), top_p=torch.where(i % 2 == 0, 1.0, 0.8), min_p=torch.where(i % 11 == 0, 0.1, 0.0))
    got = sample(x, u, **s)
    pieces = [sample(x[a:a + 500], u[a:a + 500], **{k: v[a:a + 500] for k, v in s.items()}) for a in range(0, B, 500)]
    assert torch.equal(got, torch.cat(pieces))
    at = torch.tensor([0, 1, 2, 1023, 1024, B - 2, B - 1]) if B < 70000 else torch.tensor([0, 65534, 65535, 65536, B - 1])
    check(x[at.cuda()].cpu(), u[at.cuda()], got[at.cuda()], **{k: v[at.cuda()] for k, v in s.items()})


def test_sums_that_fill_the_bins_and_more_candidates_than_there_is_room_for():
    """All elements within one bin: more of them than are looked at one by one (8192) or sorted (1024)."""
    from gaac_amd import sample
    require_gpu()
    for V in (900, 1100, 5000, 8192, 8300, 20000, 70000):
        x = 3 + torch.rand(2, V, generator=torch.Generator().manual_seed(V)) * 0.02
        u = torch.tensor([0.3, 0.95])
        for s in (dict(top_p=0.5), dict(top_k=V // 2), dict(top_k=V - 3, top_p=0.9), dict(top_p=0.7, min_p=0.99), dict(top_k=700, top_p=0.3)):
            for dtype in TYPES: check(x.to(dtype), u, sample(x.to(dtype).cuda(), u.cuda(), **s), **s)


@pytest.mark.parametrize("kind", ["model", "few values", "flat"])
@pytest.mark.parametrize("k", [1, 2, 3, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1024, 1025, 2048, 8192, 8193])
def test_as_many_candidates_as_are_put_in_order_at_a_time(k, kind):
    """A wave's, a block's and two for each thread; rows of one segment and of several; equal numbers on both sides of the limit."""
    from gaac_amd import sample
    require_gpu()
    for V in (4000, 9001):
        for i, s in enumerate((dict(top_k=k), dict(top_k=k, top_p=0.8, temperature=3.0), dict(top_k=k, top_p=0.97, min_p=0.05, temperature=1.5))):
            x, u = logits(3, V, torch.float32, 7 * k + i, kind)
            check(x, u, sample(x.cuda(), u.cuda(), **s), **s)


def test_every_token_of_a_short_list_comes():
    """Random numbers all along a row's running sum: of lists of up to 64 and of more, at the ends of the vocabulary as well."""
    from gaac_amd import sample
    require_gpu()
    for V, k in ((4000, 40), (20000, 64), (20000, 90), (1048560, 64)):
        x = torch.full((1, V), -math.inf)
        at = torch.cat([torch.tensor([0, 1, V - 2, V - 1]), torch.randperm(V - 4, generator=torch.Generator().manual_seed(k))[:k + 20] + 2])
        x[0, at] = torch.randn(len(at), generator=torch.Generator().manual_seed(V)) * 0.5
        u = (torch.arange(97) + 0.5) / 97
        rows, s = x.cuda().expand(97, V), dict(top_k=k)
        check(x.expand(97, V), u, sample(rows, u.cuda(), **s), **s)
