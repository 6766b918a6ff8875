"""Norms and rotation of queries and keys on the GPU against their definition in 64 bits."""
import pytest
import torch

import operators_ref as R
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(N, n_q, n_kv, D, rot, dtype, norm, max_pos=500, seed=0, per_head=False):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(N, n_q + 2 * n_kv, D, generator=g) * torch.exp2(torch.rand(1, n_q + 2 * n_kv, D, generator=g) * 4 - 2)).to(dtype).cuda()
    w = [(torch.rand(*((h, D) if per_head else (D,)), generator=g) + 0.5).to(dtype).cuda() if norm else None for h in (n_q, n_kv)]
    pos = torch.randint(0, max_pos, (N,), generator=g).cuda()
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * 10000.0 ** -(torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return qkv[:, :n_q], qkv[:, n_q:n_q + n_kv], w, pos, ang.cos().float().cuda(), ang.sin().float().cuda()


def check(got, x, w, pos, cos, sin, interleaved, eps):
    ref, tol = R.norm_rope(x, w, cos[pos.long()], sin[pos.long()], interleaved, eps)
    assert got.dtype == x.dtype and got.is_contiguous() and got.shape == x.shape
    err = (got.double().cpu() - ref).abs()
    assert (err <= tol).all(), f"{(err / tol).max():.3g} of the bound"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 48), (256, 256), (256, 16), (256, 192)])
@pytest.mark.parametrize("dtype", TYPES)
def test_against_the_definition(dtype, D, rot, norm, interleaved):
    from gaac_amd import qk_norm_rope
    require_gpu()
    q, k, w, pos, cos, sin = make(37, 6, 2, D, rot, dtype, norm)
    for x, weight, got in zip((q, k), w, qk_norm_rope(q, k, pos, cos, sin, *w, eps=1e-5, interleaved=interleaved)): check(got, x, weight, pos, cos, sin, interleaved, 1e-5)


@pytest.mark.parametrize("N,n_q,n_kv", [(1, 1, 1), (1, 32, 8), (2, 3, 1), (5, 40, 8), (64, 8, 8), (333, 13, 1), (2000, 32, 8), (9001, 4, 2)])
def test_sizes(N, n_q, n_kv):
    from gaac_amd import qk_norm_rope
    require_gpu()
    q, k, w, pos, cos, sin = make(N, n_q, n_kv, 128, 128, torch.bfloat16, True)
    for x, weight, got in zip((q, k), w, qk_norm_rope(q, k, pos.int(), cos, sin, *w)): check(got, x, weight, pos, cos, sin, False, 1e-6)


def test_a_weight_for_each_head():
    from gaac_amd import qk_norm_rope
    require_gpu()
    q, k, w, pos, cos, sin = make(20, 6, 3, 128, 128, torch.bfloat16, True, per_head=True)
    for x, weight, got in zip((q, k), w, qk_norm_rope(q, k, pos, cos, sin, *w)): check(got, x, weight, pos, cos, sin, False, 1e-6)
    got = qk_norm_rope(q, k, pos, cos, sin, w[0], w[1][0])      # one for each query head, one for all keys
    check(got[1], k, w[1][0], pos, cos, sin, False, 1e-6)


def test_without_weights_it_is_the_rotation_in_separate_operations():
    """Bit for bit x1 cos - x2 sin, x2 cos + x1 sin with each product and sum rounded: what a decode loop of torch operations computes."""
    from gaac_amd import qk_norm_rope
    require_gpu()
    def separate(x, c, s):
        a, b, c, s = x[..., :64].float(), x[..., 64:].float(), c[:, None], s[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)
    for dtype in TYPES:
        q, k, _, pos, cos, sin = make(300, 5, 2, 128, 128, dtype, False)
        for x, got in zip((q, k), qk_norm_rope(q, k, pos, cos, sin)): assert torch.equal(got, separate(x, cos[pos], sin[pos]))


@pytest.mark.parametrize("layout", ["head-major", "odd offset", "every other channel", "expanded"])
def test_layouts(layout):
    from gaac_amd import qk_norm_rope
    require_gpu()
    q, k, w, pos, cos, sin = make(21, 4, 2, 128, 128, torch.float16, True)
    if layout == "head-major": q, k = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k))
    elif layout == "odd offset": q, k = (torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape) for x in (q, k))
    elif layout == "every other channel": q, k = (x.repeat_interleave(2, -1)[..., ::2] for x in (q, k))
    else: q, k = q[:1].expand(21, -1, -1), k[:, :1].expand(-1, 2, -1)
    tables = cos.t().contiguous().t(), torch.cat([sin.flatten()[:1], sin.flatten()])[1:].view(sin.shape)
    both = torch.stack([pos, pos], 1)[:, 0]
    for x, weight, got in zip((q, k), w, qk_norm_rope(q, k, both, *tables, *w)): check(got, x, weight, pos, cos, sin, False, 1e-6)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rot", [128, 32])
def test_a_position_outside_the_tables_is_nan_and_no_other_token_is(rot, norm):
    from gaac_amd import qk_norm_rope
    require_gpu()
    q, k, w, pos, cos, sin = make(40, 4, 2, 128, rot, torch.bfloat16, norm, max_pos=50)
    want = qk_norm_rope(q, k, pos, cos, sin, *w)
    bad = pos.clone()
    bad[3], bad[17], bad[39] = 50, -1, 2 ** 40
    for got, ref in zip(qk_norm_rope(q, k, bad, cos, sin, *w), want):
        hit = torch.tensor([i in (3, 17, 39) for i in range(40)])
        assert got[hit].isnan().all() and torch.equal(got[~hit], ref[~hit])


def test_rows_of_zeros_infinities_and_nan():
    """Zeros stay zeros (eps keeps the quotient finite), a NaN or an infinity stays in its head."""
    from gaac_amd import qk_norm_rope
    require_gpu()
    q, k, w, pos, cos, sin = make(9, 4, 2, 128, 128, torch.bfloat16, True)
    q = q.clone()
    q[2, 1] = 0; q[3, 0, 5] = float("nan"); q[4, 3, 100] = float("inf")
    got, _ = qk_norm_rope(q, k, pos, cos, sin, *w)
    assert (got[2, 1] == 0).all() and got[3, 0].isnan().all() and got[4, 3].isnan().any()
    keep = torch.ones(9, 4, dtype=torch.bool)
    keep[3, 0] = keep[4, 3] = False
    assert not got[keep].isnan().any()


def test_no_tokens_and_a_captured_call():
    from gaac_amd import qk_norm_rope
    require_gpu()
    q, k, w, pos, cos, sin = make(6, 4, 2, 128, 128, torch.bfloat16, True)
    assert qk_norm_rope(q[:0], k[:0], pos[:0], cos, sin, *w)[0].shape == (0, 4, 128)
    want = qk_norm_rope(q, k, pos, cos, sin, *w)
    buf = pos.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g): got = qk_norm_rope(q, k, buf, cos, sin, *w)
    for step in range(4):
        buf.copy_((pos + step) % 500)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) == (step == 0)
        for a, b in zip(got, qk_norm_rope(q, k, (pos + step) % 500, cos, sin, *w)): assert torch.equal(a, b)
