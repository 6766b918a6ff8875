"""Refusals of the 4-bit cache, norm + rotation and sampling, and their sizes, without a GPU: every call that cannot be made raises before anything is launched."""
import pytest
import torch

from gaac_amd import FP4KVCache, qk_norm_rope, sample
from gaac_amd import _lib
from gaac_amd.fp4_cache import choose_nsplit

BF = torch.bfloat16


def test_sizes_of_the_cache():
    assert FP4KVCache.bytes_per_slot(8, 65536) == 8 * 2048 * 4352 + 4 and FP4KVCache.bytes_per_slot(1, 1) == 4352 + 4
    assert [choose_nsplit(*x) for x in ((1, 8, 65536), (1, 8, 100), (1, 8, 2000), (16, 8, 65536), (32, 8, 6000), (300, 8, 65536), (1, 1, 10 ** 6))] == [32, 1, 15, 4, 1, 2, 128]
    assert [choose_nsplit(1, 1, S, G) for S in (8192, 32768, 131072, 10 ** 6) for G in (1, 4, 16)] == [16, 16, 16, 32, 32, 32, 64, 64, 32, 128, 128, 64]
    for bad in ((0, 8, 64), (1, 0, 64), (1, 8, 0)):
        with pytest.raises(RuntimeError, match="at least 1"): FP4KVCache(*bad, device="cpu")


def test_cache_calls_that_are_refused():
    c = FP4KVCache(2, 4, 64, device="cpu")
    x = torch.zeros(10, 4, 128, dtype=BF)
    for k, v in ((x.float(), x), (x, x.half()), (x, x[:5]), (x[:, :3], x[:, :3]), (x[..., :64], x[..., :64]), (x[0], x[0])):
        with pytest.raises(RuntimeError, match="prefill expects k, v bf16"): c.prefill(0, k, v)
        with pytest.raises(RuntimeError, match="append expects k, v bf16"): c.append(torch.zeros(10, dtype=torch.int32), k, v)
    for slot in (-1, 2):
        with pytest.raises(RuntimeError, match="slot in 0..1"): c.prefill(slot, x, x)
        with pytest.raises(RuntimeError, match="slot in 0..1"): c.decompress(slot)
    long = torch.zeros(65, 4, 128, dtype=BF)
    with pytest.raises(RuntimeError, match="prompt has 65 tokens, a slot holds 64"): c.prefill(0, long, long)
    for slots in (torch.zeros(10, dtype=torch.int64), torch.zeros(9, dtype=torch.int32), torch.zeros(10, 1, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match=r"slots int32 \[B\]"): c.append(slots, x, x)
        with pytest.raises(RuntimeError, match=r"slots int32 \[B\]"): c.attention(x.repeat(1, 2, 1), slots, 1.0)
    slots = torch.zeros(10, dtype=torch.int32)
    for q in (x.float(), x[..., :64], x[0]):
        with pytest.raises(RuntimeError, match="attention expects q bf16"): c.attention(q, slots, 1.0)
    for n_q in (0, 3, 5, 68):
        with pytest.raises(RuntimeError, match="GQA group size must be 1..16"): c.attention(torch.zeros(10, n_q, 128, dtype=BF), slots, 1.0)
    with pytest.raises(RuntimeError, match="at least one split"): c.attention(x, slots, 1.0, nsplit=0)
    for call in (lambda: c.prefill(0, x, x), lambda: c.append(slots, x, x), lambda: c.attention(x, slots, 1.0)):      # all in order but for the device
        with pytest.raises(RuntimeError, match="no CPU path"): call()


def test_capacity_words_name_what_was_lost():
    c = FP4KVCache(2, 4, 64, device="cpu")
    c.check_capacity()
    for bits, texts in ((1, ["token capacity"]), (2, ["twice"]), (4, ["does not exist"]), (7, ["token capacity", "twice", "does not exist"])):
        with pytest.raises(RuntimeError) as e: c.check_capacity(bits)
        assert all(t in str(e.value) for t in texts)


def test_rotations_that_are_refused():
    q, k, pos, cos = torch.zeros(5, 8, 128), torch.zeros(5, 2, 128), torch.zeros(5, dtype=torch.int64), torch.zeros(10, 64)
    for a, b in ((q, k.half()), (q.double(), k.double()), (q[:4], k), (q[..., :64], k), (q[0], k), (q[:, :0], k), (q[..., :96], k[..., :96])):
        with pytest.raises(RuntimeError, match="qk_norm_rope expects"): qk_norm_rope(a, b, pos, cos, cos)
    for p in (pos.float(), pos[:4], pos[:, None]):
        with pytest.raises(RuntimeError, match="positions"): qk_norm_rope(q, k, p, cos, cos)
    for c, s in ((cos.half(), cos), (cos, cos[:9]), (cos[:0], cos[:0]), (cos[:, :4], cos[:, :4]), (cos[:, :12], cos[:, :12]), (torch.zeros(10, 72), torch.zeros(10, 72)), (cos[0], cos[0])):
        with pytest.raises(RuntimeError, match="cos, sin"): qk_norm_rope(q, k, pos, c, s)
    w = torch.ones(128)
    with pytest.raises(RuntimeError, match="for both"): qk_norm_rope(q, k, pos, cos, cos, w)
    with pytest.raises(RuntimeError, match="for both"): qk_norm_rope(q, k, pos, cos, cos, None, w)
    for a, b in ((w.half(), w), (w, w[:64]), (torch.ones(2, 128), w), (w, torch.ones(8, 128))):
        with pytest.raises(RuntimeError, match="weights"): qk_norm_rope(q, k, pos, cos, cos, a, b)
    with pytest.raises(RuntimeError, match="no CPU path"): qk_norm_rope(q, k, pos, cos, cos, w, w)


def test_samples_that_are_refused():
    x, u = torch.zeros(4, 100), torch.zeros(4)
    for bad in (x.double(), x[0], x[:, :0], torch.zeros(1).expand(2, 1 << 20)):
        with pytest.raises(RuntimeError, match="sample expects logits"): sample(bad, u)
    for bad in (u.double(), u[:3], u[:, None]):
        with pytest.raises(RuntimeError, match="sample expects u"): sample(x, bad)
    for name, bad in (("temperature", u.double()), ("temperature", u[:3]), ("top_k", u), ("top_k", torch.zeros(4, dtype=torch.int64)), ("top_p", u[:, None]), ("min_p", u.half())):
        with pytest.raises(RuntimeError, match=f"sample expects {name}"): sample(x, u, **{name: bad})
    with pytest.raises(RuntimeError, match="no CPU path"): sample(x, u)


@pytest.mark.parametrize("name,args,message", [
    ("gaac_fp4_store", [16, 16, 128, 1024, 128, 1024, 65, 8, 2, 16, 16, None], "bad sizes"),
    ("gaac_fp4_store", [16, 18, 128, 1024, 128, 1024, 64, 8, 2, 16, 16, None], "16-byte aligned"),
    ("gaac_fp4_store", [16, 16, 127, 1024, 128, 1024, 64, 8, 2, 16, 16, None], "16-byte aligned"),
    ("gaac_fp4_load", [16, 0, 8, 2, 16, 16, 128, 1024, 128, 1024, None], "bad sizes"),
    ("gaac_fp4_load", [16, 64, 8, 2, 16, 16, 128, 1020, 128, 1024, None], "16-byte aligned"),
    ("gaac_fp4_append", [16, 4, 2, 8, 16, 16, 1024, 128, 1024, 128, 16, 2, 65, 16, 16, None], "bad sizes"),
    ("gaac_fp4_append", [16, 4, 2, 8, 16, 17, 1024, 128, 1024, 128, 16, 2, 64, 16, 16, None], "16-byte aligned"),
    ("gaac_fp4_attn", [16, 16, 16, 2, 2, 64, 16, 1, 9, 8, 1.0, 1, None, None, 16, None], "GQA group"),
    ("gaac_fp4_attn", [16, 16, 16, 2, 2, 64, 16, 1, 136, 8, 1.0, 1, None, None, 16, None], "GQA group"),
    ("gaac_fp4_attn", [16, 16, 16, 2, 2, 64, 16, 1, 8, 8, 1.0, 2, None, None, 16, None], "needs partials"),
    ("gaac_fp4_attn", [16, 16, 16, 2, 2, 64, 16, 1, 8, 8, 1.0, 0, None, None, 16, None], "bad sizes"),
    ("gaac_fp4_attn", [16, 16, 16, 2, 2, 64, 24, 1, 8, 8, 1.0, 1, None, None, 16, None], "16-byte aligned"),
    ("gaac_qk_norm_rope", [3, 16, 16, 1, 1, 1, 1, 1, 1, 1, 128, 128, None, None, 0, 0, 1e-6, 16, 1, 16, 16, 1, 0, 16, 16, None], "type must be"),
    ("gaac_qk_norm_rope", [0, 16, 16, 8, 8, 8, 8, 1, 1, 1, 96, 96, None, None, 0, 0, 1e-6, 16, 1, 16, 16, 1, 0, 16, 16, None], "head_dim must be"),
    ("gaac_qk_norm_rope", [0, 16, 16, 8, 8, 8, 8, 1, 1, 1, 128, 136, None, None, 0, 0, 1e-6, 16, 1, 16, 16, 1, 0, 16, 16, None], "head_dim must be"),
    ("gaac_qk_norm_rope", [0, 16, 16, 8, 8, 8, 8, 0, 1, 1, 128, 128, None, None, 0, 0, 1e-6, 16, 1, 16, 16, 1, 0, 16, 16, None], "bad sizes"),
    ("gaac_qk_norm_rope", [0, 16, 16, 8, 8, 8, 8, 1, 1, 1, 128, 128, 16, None, 0, 0, 1e-6, 16, 1, 16, 16, 1, 0, 16, 16, None], "for both"),
    ("gaac_qk_norm_rope", [0, 16, 16, 8, 4, 8, 8, 1, 1, 1, 128, 128, None, None, 0, 0, 1e-6, 16, 1, 16, 16, 1, 0, 16, 16, None], "16-byte aligned"),
    ("gaac_sample", [0, 16, 100, 0, 100, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, 16, 1 << 30, 16, None], "bad sizes"),
    ("gaac_sample", [0, 16, 100, 1, 1 << 20, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, 16, 1 << 30, 16, None], "bad sizes"),
    ("gaac_sample", [0, 17, 100, 1, 100, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, 16, 1 << 30, 16, None], "not aligned"),
    ("gaac_sample", [0, 16, 5000, 2, 5000, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, 16, 2 * (32 + 90128) - 1, 16, None], "work memory"),
    ("gaac_sample", [0, 16, 5000, 1, 5000, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, 20, 1 << 20, 16, None], "work memory"),
    ("gaac_sample", [0, 16, 5000, 1, 5000, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, None, 1 << 20, 16, None], "work memory"),
])
def test_the_library_refuses_before_it_launches(name, args, message):
    with pytest.raises(RuntimeError, match=f"{name} failed .*{message}"): _lib.call(name, *args)


def test_gradients_are_not_lost_without_a_word():
    x, pos, cos, w = torch.zeros(5, 2, 128, dtype=BF), torch.zeros(5, dtype=torch.int64), torch.zeros(10, 64), torch.ones(128, dtype=BF)
    need = lambda t: t.clone().requires_grad_()
    c = FP4KVCache(2, 2, 64, device="cpu")
    calls = (lambda t: qk_norm_rope(t(x), x, pos, cos, cos), lambda t: qk_norm_rope(x, t(x), pos, cos, cos, w, w), lambda t: qk_norm_rope(x, x, pos, cos, cos, t(w), w), lambda t: qk_norm_rope(x, x, pos, cos, cos, w, t(w)),
             lambda t: c.attention(t(x), torch.zeros(5, dtype=torch.int32), 1.0))
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward pass"): call(need)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"): call(need)
