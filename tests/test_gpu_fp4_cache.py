"""The 4-bit slot cache on the GPU: what it holds against its definition, bit for bit; attention over it against attention in 64 bits over those values."""
import math

import pytest
import torch

import operators_ref as R
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
D = 128


def rows(L, n_kv, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(L, n_kv, D, generator=g) * torch.exp2((torch.rand(1, n_kv, D, generator=g) * 2 - 1) * spread)
    return x.to(torch.bfloat16).cuda()


def cache(*args):
    from gaac_amd import FP4KVCache
    return FP4KVCache(*args)


def same(a, b):
    """Equal as numbers, NaN where NaN."""
    a, b = a.double().cpu(), b.double().cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def check(out, q, held, scale):
    """out [B, n_q, D] against attention in 64 bits over held: per row (k, v) values or None (0)."""
    out = out.double().cpu()
    for b, kv in enumerate(held):
        if kv is None or kv[0].shape[0] == 0:
            assert (out[b] == 0).all(), f"row {b}"
            continue
        ref, tol = R.attention(q[b], *kv, scale)
        err = (out[b] - ref).abs()
        assert (err <= tol).all(), f"row {b}: {(err / tol).max():.3g} of the bound"


# ---------------------------------------------------------------------------------------------------- what is held
@pytest.mark.parametrize("n_kv", [1, 3, 8])
@pytest.mark.parametrize("L", [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 333])
def test_a_prompt_is_held_by_definition(L, n_kv):
    require_gpu()
    k, v = rows(L, n_kv, 1), rows(L, n_kv, 2)
    c = cache(3, n_kv, 350)
    c.prefill(1, k, v)
    dk, dv = c.decompress(1)
    assert same(dk, R.stored(k)) and same(dv, R.stored(v))
    assert c.lens.tolist() == [0, L, 0] and not c.data[:n_kv].any() and not c.data[2 * n_kv:].any()


def test_every_bf16_value_in_blocks_of_every_maximum():
    """All 65536 patterns, each in a block whose maximum is itself, up to 8 times or up to 2^20 times as large; NaN, infinities, subnormals, both zeros."""
    require_gpu()
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    for up in (1.0, 1.7, 3.0, 5.5, 8.0, 2.0 ** 20):
        b = x[:, None].repeat(1, 32)
        b[:, 7] = (x.float() * up).clamp(-3.38e38, 3.38e38).to(torch.bfloat16)
        t = b.reshape(-1, 4, D).contiguous().cuda()
        c = cache(1, 4, t.shape[0])
        c.prefill(0, t, t.flip(0).contiguous())
        k, v = c.decompress(0)
        assert same(k, R.stored(t)) and same(v, R.stored(t.flip(0)))


def test_nearest_codes_ties_to_even_and_exponents():
    """A block by hand: maximum 6.5 < 7 keeps E = 0, 7 raises it.  (5.01 is 5 in bf16, whose neighbours are 1/32 apart there: a tie.)"""
    require_gpu()
    x = torch.zeros(2, 1, D)
    x[0, 0, :16] = torch.tensor([6.5, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, -0.25, -0.75, -2.5, -5.0, 0.5, -6.0])
    x[1, 0, :4] = torch.tensor([7.0, 0.5, 1.5, 2.5])
    t = x.to(torch.bfloat16).cuda()
    c = cache(1, 1, 32)
    c.prefill(0, t, t)
    for y in c.decompress(0):
        y = y.float().cpu()
        assert y[0, 0, :16].tolist() == [6.0, 0.0, 0.5, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 4.0, -0.0, -1.0, -2.0, -4.0, 0.5, -6.0]
        assert y[1, 0, :4].tolist() == [8.0, 0.0, 2.0, 2.0]
        assert (y[:, 0, 32:] == 0).all()


def test_appended_tokens_are_held_as_a_prompts_are():
    """Tokens that arrive one by one, in rows of different lengths and with rows left out, leave byte for byte what a prompt of the same tokens leaves."""
    require_gpu()
    n_kv, starts, steps = 3, [0, 1, 15, 31, 40], 70
    B = len(starts)
    k, v = [rows(s + steps, n_kv, 10 + i) for i, s in enumerate(starts)], [rows(s + steps, n_kv, 20 + i) for i, s in enumerate(starts)]
    a, b = cache(B + 1, n_kv, 128), cache(B + 1, n_kv, 128)
    slots = [4, 0, 3, 1, 5]
    for i, s in enumerate(starts):
        a.prefill(slots[i], k[i][:s], v[i][:s])
    held = list(starts)
    for step in range(steps):
        out = [step % 7 == i for i in range(B)]      # rows that pause
        m = torch.tensor([-1 if out[i] else slots[i] for i in range(B)], dtype=torch.int32, device="cuda")
        a.append(m, torch.stack([k[i][held[i]] for i in range(B)]), torch.stack([v[i][held[i]] for i in range(B)]))
        held = [h + (not o) for h, o in zip(held, out)]
    for i in range(B): b.prefill(slots[i], k[i][:held[i]], v[i][:held[i]])
    a.check_capacity()
    assert torch.equal(a.lens, b.lens) and torch.equal(a.data, b.data)


@pytest.mark.parametrize("layout", ["view of a fused projection", "head-major", "odd offset", "expanded"])
def test_rows_are_read_through_strides(layout):
    require_gpu()
    n_kv, L = 4, 45
    if layout == "view of a fused projection":
        x = rows(L, 6 + 2 * n_kv, 3)
        k, v = x[:, 6:6 + n_kv], x[:, 6 + n_kv:]
    elif layout == "head-major":
        k, v = rows(n_kv, L, 4).transpose(0, 1), rows(n_kv, L, 5).transpose(0, 1)
    elif layout == "odd offset":      # rows that are not 16-byte aligned
        k, v = (rows(L, n_kv + 1, s).flatten()[3:3 + L * n_kv * D].view(L, n_kv, D) for s in (6, 7))
    else:
        k, v = rows(1, n_kv, 8).expand(L, -1, -1), rows(L, 1, 9).expand(-1, n_kv, -1)
    a, b = cache(2, n_kv, 64), cache(2, n_kv, 64)
    a.prefill(1, k, v); b.prefill(1, k.contiguous(), v.contiguous())
    assert torch.equal(a.data, b.data)
    s = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    a.append(s, k[:2], v[:2]); b.append(s, k[:2].contiguous(), v[:2].contiguous())
    assert torch.equal(a.data, b.data) and a.lens.tolist() == [1, L + 1]


def test_rows_that_cannot_be_added_are_left_out_and_reported():
    require_gpu()
    n_kv = 2
    k, v = rows(64, n_kv, 1), rows(64, n_kv, 2)
    def fresh():
        c = cache(3, n_kv, 64)
        c.prefill(0, k[:40], v[:40]); c.prefill(1, k, v)
        return c
    for slots, bit, message, lens in (([1, 0], 1, "token capacity", [41, 64, 0]), ([2, 0, 2], 2, "twice", [41, 64, 1]), ([3, 0], 4, "does not exist", [41, 64, 0]), ([2 ** 31 - 1, -5], 4, "does not exist", [40, 64, 0])):
        c = fresh()
        before = c.data.clone()
        c.append(torch.tensor(slots, dtype=torch.int32, device="cuda"), k[:len(slots)], v[:len(slots)])
        assert int(c.overflow) == bit and c.lens.tolist() == lens
        with pytest.raises(RuntimeError, match=message): c.check_capacity()
        assert torch.equal(c.data[n_kv:2 * n_kv], before[n_kv:2 * n_kv])
        want = fresh()
        for s in sorted(set(slots) & {0, 2}):      # what the rows that count leave
            i = slots.index(s)
            want.append(torch.tensor([s], dtype=torch.int32, device="cuda"), k[i:i + 1], v[i:i + 1])
        assert torch.equal(c.data, want.data)


def test_lengths_that_a_caller_set_wrongly():
    """lens is a tensor of the caller's to write (to drop tokens): below 0 counts as an empty slot that takes no token, above the capacity as a full one."""
    require_gpu()
    n_kv, L = 2, 64
    k, v = rows(L, n_kv, 1), rows(L, n_kv, 2)
    slots = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    for nsplit in (1, 3):
        c = cache(3, n_kv, L)
        for s in range(3): c.prefill(s, k, v)
        held = c.decompress(1)
        c.lens.copy_(torch.tensor([-40, 64, 2 ** 31 - 1], dtype=torch.int32))
        check(c.attention(q, slots, D ** -0.5, nsplit=nsplit), q, [None, held, held], D ** -0.5)
        before = c.data.clone()
        c.append(slots, k[:3], v[:3])
        assert int(c.overflow) == 1 and torch.equal(c.data, before) and c.lens.tolist() == [-40, 64, 2 ** 31 - 1]


# ---------------------------------------------------------------------------------------------------- attention
HEADS = [(8, 4), (4, 6), (1, 16), (16, 1), (2, 5), (3, 13), (1, 14), (1, 15)]


@pytest.mark.parametrize("n_kv,G", HEADS)
@pytest.mark.parametrize("nsplit", [None, 1, 2, 7])
def test_attention_over_lengths_at_the_edges_of_tiles(n_kv, G, nsplit):
    require_gpu()
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 255, 256, 257, 300]
    c = cache(len(lens), n_kv, 320)
    held = []
    for i, L in enumerate(lens):
        k, v = rows(L, n_kv, 30 + i), rows(L, n_kv, 60 + i)
        c.prefill(i, k, v)
        held.append((R.stored(k), R.stored(v)))
    order = [5, 0, -1, 15, 3, 9, 1, 2, 8, 14, 13, 4, 6, 7, 10, 11, 12, -1, 15, 15]      # padded rows, a slot three times
    q = torch.randn(len(order), n_kv * G, D, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).cuda()
    out = c.attention(q, torch.tensor(order, dtype=torch.int32, device="cuda"), D ** -0.5, nsplit=nsplit)
    check(out, q, [None if s < 0 else held[s] for s in order], D ** -0.5)


@pytest.mark.parametrize("L,n_kv,G,nsplit", [(1, 1, 1, None), (1000, 8, 4, None), (5000, 2, 8, None), (5000, 2, 8, 1), (5000, 1, 3, 256), (33, 8, 4, 16), (20011, 1, 16, None), (4097, 8, 1, 33)])
def test_attention_of_a_single_row(L, n_kv, G, nsplit):
    require_gpu()
    k, v = rows(L, n_kv, 1), rows(L, n_kv, 2)
    c = cache(2, n_kv, L)
    c.prefill(1, k, v)
    q = torch.randn(1, n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    out = c.attention(q, torch.tensor([1], dtype=torch.int32, device="cuda"), D ** -0.5, max_len=L, nsplit=nsplit)
    check(out, q, [(R.stored(k), R.stored(v))], D ** -0.5)


@pytest.mark.parametrize("B", [63, 64, 65, 130, 300])
@pytest.mark.parametrize("nsplit", [None, 1, 2, 5])
def test_attention_of_large_batches(B, nsplit):
    """More rows than lanes: the rows' splits are counted in rounds of 64."""
    require_gpu()
    n_kv, G = 2, 2
    lens = [(37 * i * i + 11 * i) % 400 for i in range(B)]
    lens[B // 2] = 2000
    c = cache(B, n_kv, 2000)
    held = []
    for i, L in enumerate(lens):
        k, v = rows(L, n_kv, i), rows(L, n_kv, 1000 + i)
        c.prefill(i, k, v)
        held.append((R.stored(k), R.stored(v)))
    q = torch.randn(B, n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    check(c.attention(q, torch.arange(B, dtype=torch.int32, device="cuda"), D ** -0.5, nsplit=nsplit), q, held, D ** -0.5)


@pytest.mark.parametrize("scale", [D ** -0.5, 1.0, -0.3, 0.0, 4.0, 1e-6])
def test_scales(scale):
    require_gpu()
    L, n_kv, G = 700, 2, 4
    k, v = rows(L, n_kv, 1), rows(L, n_kv, 2)
    c = cache(1, n_kv, L)
    c.prefill(0, k, v)
    q = torch.randn(1, n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    for nsplit in (1, 4): check(c.attention(q, torch.zeros(1, dtype=torch.int32, device="cuda"), scale, nsplit=nsplit), q, [(R.stored(k), R.stored(v))], scale)


def test_scores_that_rise_all_along_the_row():
    """The running maximum is raised again and again, and the last token holds all of the weight; then the other way round."""
    require_gpu()
    L, n_kv, G = 999, 1, 4
    k = torch.zeros(L, n_kv, D)
    k[:, :, 0] = torch.linspace(-200, 200, L)[:, None]
    v = rows(L, n_kv, 2)
    q = torch.ones(2, n_kv * G, D).to(torch.bfloat16).cuda()
    c = cache(2, n_kv, L)
    for i, kk in enumerate((k, k.flip(0))): c.prefill(i, kk.to(torch.bfloat16).cuda(), v)
    for nsplit in (1, 3):
        out = c.attention(q, torch.arange(2, dtype=torch.int32, device="cuda"), 1.0, nsplit=nsplit)
        check(out, q, [(R.stored(kk.to(torch.bfloat16)), R.stored(v)) for kk in (k, k.flip(0))], 1.0)


def test_values_of_every_size():
    """Values of 2^100 and of 2^-100 beside ordinary ones: weights are not scaled into the values' range or out of it."""
    require_gpu()
    L, n_kv, G = 100, 1, 2
    for size in (2.0 ** 100, 2.0 ** -100, 2.0 ** -118):
        k, v = rows(L, n_kv, 1), (rows(L, n_kv, 2).float() * size).to(torch.bfloat16)
        c = cache(1, n_kv, L)
        c.prefill(0, k, v)
        q = torch.randn(1, n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
        check(c.attention(q, torch.zeros(1, dtype=torch.int32, device="cuda"), D ** -0.5), q, [(R.stored(k), R.stored(v))], D ** -0.5)


@pytest.mark.parametrize("L", [1, 5, 16, 17, 33, 100, 300])
@pytest.mark.parametrize("nsplit", [1, 3])
def test_what_an_earlier_sequence_left_behind_the_end_does_not_count(L, nsplit):
    """The slot was full of NaN, infinities and the largest numbers; a shorter prompt, and then tokens, take its place."""
    require_gpu()
    n_kv, G = 2, 4
    c = cache(1, n_kv, 320)
    bad = torch.full((320, n_kv, D), math.nan)
    bad[::3] = math.inf; bad[1::3] = 3.3e38
    c.prefill(0, bad.to(torch.bfloat16).cuda(), bad.to(torch.bfloat16).cuda())
    k, v = rows(L + 3, n_kv, 1), rows(L + 3, n_kv, 2)
    q = torch.randn(1, n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    slots = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.prefill(0, k[:L], v[:L])
    for i in range(4):
        check(c.attention(q, slots, D ** -0.5, nsplit=nsplit), q, [(R.stored(k[:L + i]), R.stored(v[:L + i]))], D ** -0.5)
        if i < 3: c.append(slots, k[L + i:L + i + 1], v[L + i:L + i + 1])


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("nsplit", [1, 4])
def test_a_nan_that_is_held_reaches_its_rows_and_no_others(where, nsplit):
    require_gpu()
    L, n_kv, G = 200, 2, 4
    k, v = rows(L, n_kv, 1), rows(L, n_kv, 2)
    x = k if where == "k" else v
    bad = x.clone()
    bad[77, 1, 40] = math.nan      # head 1, second block
    c = cache(2, n_kv, L)
    c.prefill(0, *((bad, v) if where == "k" else (k, bad)))
    c.prefill(1, k, v)
    q = torch.randn(2, n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    out = c.attention(q, torch.arange(2, dtype=torch.int32, device="cuda"), D ** -0.5, nsplit=nsplit)
    hit = torch.zeros(2, n_kv * G, D, dtype=torch.bool)
    hit[0, G:, slice(None) if where == "k" else slice(32, 64)] = True
    assert torch.equal(out.isnan().cpu(), hit)
    clean = c.attention(q.flip(0).contiguous(), torch.ones(2, dtype=torch.int32, device="cuda"), D ** -0.5, nsplit=nsplit)
    check(clean, q.flip(0), [(R.stored(k), R.stored(v))] * 2, D ** -0.5)


@pytest.mark.parametrize("nsplit", [1, 2])
def test_a_slot_that_does_not_exist_is_nan(nsplit):
    require_gpu()
    c = cache(2, 2, 64)
    k, v = rows(50, 2, 1), rows(50, 2, 2)
    c.prefill(0, k, v)
    q = torch.ones(4, 4, D, dtype=torch.bfloat16, device="cuda")
    out = c.attention(q, torch.tensor([0, 2, -1, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), D ** -0.5, nsplit=nsplit)
    assert out[1].isnan().all() and out[3].isnan().all() and (out[2] == 0).all()
    check(out[:1], q, [(R.stored(k), R.stored(v))], D ** -0.5)


def test_a_cache_of_more_than_four_gibibytes():
    """Offsets beyond 32 bits: the last slot of a cache of 4.6 GiB against a small one, byte for byte, and the same attention."""
    require_gpu()
    n_kv, L = 8, 1000
    big, small = cache(70, n_kv, 65536), cache(1, n_kv, 65536)
    assert big.data.numel() > 2 ** 32
    k, v = rows(L, n_kv, 1), rows(L, n_kv, 2)
    big.prefill(69, k[:-1], v[:-1]); small.prefill(0, k[:-1], v[:-1])
    at, zero = torch.tensor([69], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    big.append(at, k[-1:], v[-1:]); small.append(zero, k[-1:], v[-1:])
    assert torch.equal(big.data[69 * n_kv:], small.data) and not big.data[:8].any()
    q = torch.randn(1, 32, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    out = big.attention(q, at, D ** -0.5)
    assert torch.equal(out, small.attention(q, zero, D ** -0.5))
    for a, b in zip(big.decompress(69), (k, v)): assert same(a, R.stored(b))
    check(out, q, [(R.stored(k), R.stored(v))], D ** -0.5)


def test_two_attentions_of_one_cache_at_once():
    """Readers on two streams keep nothing in common."""
    require_gpu()
    n_kv, G, L = 4, 4, 4000
    k, v = rows(L, n_kv, 1), rows(L, n_kv, 2)
    c = cache(2, n_kv, L)
    c.prefill(0, k, v); c.prefill(1, v, k)
    q = [torch.randn(2, n_kv * G, D, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).cuda() for s in (3, 4)]
    slots = [torch.tensor(s, dtype=torch.int32, device="cuda") for s in ([0, 1], [1, 0])]
    want = [c.attention(x, s, D ** -0.5) for x, s in zip(q, slots)]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st): got[i].append(c.attention(q[i], slots[i], D ** -0.5))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]: assert torch.equal(x, want[i])


def test_a_captured_step_is_replayed():
    """append and attention in a graph; two graphs of the same shape, replayed in turn and with eager steps between, hold what eager steps hold."""
    require_gpu()
    n_kv, G, B = 2, 4, 3
    a, b = cache(B, n_kv, 256), cache(B, n_kv, 256)
    for i, L in enumerate((0, 31, 100)):
        k, v = rows(L, n_kv, i), rows(L, n_kv, 10 + i)
        a.prefill(i, k, v); b.prefill(i, k, v)
    new = [[t.cuda() for t in (torch.randn(B, n_kv * G, D).to(torch.bfloat16), torch.randn(B, n_kv, D).to(torch.bfloat16), torch.randn(B, n_kv, D).to(torch.bfloat16))] for _ in range(12)]
    slots = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    buf = [t.clone() for t in new[0]]
    a.attention(buf[0], slots, D ** -0.5, nsplit=2)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a.append(slots, buf[1], buf[2])
            out = a.attention(buf[0], slots, D ** -0.5, nsplit=2)
        graphs.append((g, out))
    for step, (q, k, v) in enumerate(new):
        b.append(slots, k, v)
        want = b.attention(q, slots, D ** -0.5, nsplit=2)
        if step % 4 == 3:
            a.append(slots, k, v)
            got = a.attention(q, slots, D ** -0.5, nsplit=2)
        else:
            for t, x in zip(buf, (q, k, v)): t.copy_(x)
            g, got = graphs[step % 2]
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"step {step}"
        assert torch.equal(a.data, b.data) and torch.equal(a.lens, b.lens)


def test_queries_and_slots_of_other_layouts():
    require_gpu()
    n_kv, G, L = 2, 4, 150
    k, v = rows(L, n_kv, 1), rows(L, n_kv, 2)
    c = cache(3, n_kv, L)
    c.prefill(2, k, v)
    x = torch.randn(3, 2 * n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    slots = torch.tensor([2, 9, 2, 9, -1, 9], dtype=torch.int32, device="cuda")[::2]
    check(c.attention(x[:, ::2], slots, D ** -0.5), x[:, ::2], [(R.stored(k), R.stored(v))] * 2 + [None], D ** -0.5)
    odd = torch.zeros(n_kv * G * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(1, n_kv * G, D)
    odd.copy_(x[:1, ::2])
    check(c.attention(odd, slots[:1], D ** -0.5), x[:1, ::2], [(R.stored(k), R.stored(v))], D ** -0.5)
    assert c.attention(x[:0, ::2], slots[:0], D ** -0.5).shape == (0, n_kv * G, D)


def test_stats_and_sizes():
    require_gpu()
    from gaac_amd import FP4KVCache
    c = cache(3, 4, 100)
    assert c.cap == 128 and FP4KVCache.bytes_per_slot(4, 100) * 3 == c.data.numel() + c.lens.numel() * 4
    c.prefill(0, rows(70, 4), rows(70, 4)); c.prefill(2, rows(5, 4), rows(5, 4))
    s = c.stats()
    assert s["tokens"] == 75 and s["bytes_used"] == 75 * 4 * 136 and s["bf16_bytes"] == 75 * 4 * 512 and abs(s["ratio"] - 512 / 136) < 1e-12


def test_a_saved_cache_is_read_as_before(tmp_path):
    require_gpu()
    n_kv, G = 2, 4
    c = cache(2, n_kv, 3000)
    k, v = rows(2500, n_kv, 1), rows(2500, n_kv, 2)
    c.prefill(1, k, v)
    q = torch.randn(1, n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    slots = torch.ones(1, dtype=torch.int32, device="cuda")
    want = c.attention(q, slots, D ** -0.5)
    torch.save(c, tmp_path / "cache.pt")
    d = torch.load(tmp_path / "cache.pt", weights_only=False)
    assert torch.equal(d.attention(q, slots, D ** -0.5), want)
    d.append(slots, k[:1], v[:1])
    assert d.lens.tolist() == [0, 2501] and c.lens.tolist() == [0, 2500]


def test_more_captured_calls_than_there_are_counters_for(monkeypatch):
    """Calls captured behind the last set of counters, or of more rows than slots, take the launch of their own that adds up the splits."""
    from gaac_amd import fp4_cache
    require_gpu()
    monkeypatch.setattr(fp4_cache, "CAPTURES", 2)
    n_kv, G, B = 2, 4, 5
    c = cache(3, n_kv, 600)
    k, v = rows(600, n_kv, 1), rows(600, n_kv, 2)
    for i, L in enumerate((600, 33, 257)): c.prefill(i, k[:L], v[:L])
    q = torch.randn(B, n_kv * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    few, many = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda"), torch.tensor([0, 0, 2, -1, 1], dtype=torch.int32, device="cuda")
    want = [c.attention(q[:3], few, D ** -0.5, nsplit=4), c.attention(q, many, D ** -0.5, nsplit=4)]
    graphs = []
    for i in range(5):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g): out = c.attention(q, many, D ** -0.5, nsplit=4) if i == 1 else c.attention(q[:3], few, D ** -0.5, nsplit=4)
        graphs.append((g, out, want[i == 1]))
    assert c._captured == 2
    for _ in range(3):
        for g, out, ref in graphs:
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ref)
            assert torch.equal(c.attention(q, many, D ** -0.5, nsplit=4), want[1])
