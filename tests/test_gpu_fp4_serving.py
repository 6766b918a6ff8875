"""The operators of a decode step together, as the decode loop runs them: norm + rotation, the 4-bit cache's writes and attention, sampling."""
import pytest
import torch

import operators_ref as R
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu


def setup(kv, qk_norm=True, n_slots=3):
    from gaac_amd.serving import DecodeRunner, ModelConfig, Weights
    dev = require_gpu()
    cfg = ModelConfig(hidden=256, n_layers=2, n_heads=8, n_kv_heads=2, ffn=512, vocab=5000, rope_theta=10000.0, max_len=512, qk_norm=qk_norm)
    w = Weights(cfg, dev, seed=1)
    if qk_norm:
        g = torch.Generator(device=dev).manual_seed(3)
        for l in w.layers:
            for name in ("q_norm", "k_norm"): l[name] = (torch.rand(128, generator=g, device=dev) + 0.5).to(torch.bfloat16)
    run = DecodeRunner(w, n_slots=n_slots, kv=kv)
    g = torch.Generator(device=dev).manual_seed(2)
    prompts = [torch.randint(0, cfg.vocab, (L,), generator=g, device=dev) for L in (200, 37, 64)]
    first = torch.stack([run.prefill(i, p).argmax() for i, p in enumerate(prompts)])
    return cfg, w, run, prompts, first


@pytest.mark.parametrize("qk_norm", [False, True])
def test_every_layer_of_a_step_against_the_definitions(qk_norm):
    """What each layer's cache holds is its definition of the K and V the layer was handed, through prompts and steps; every step's attention is that of 64 bits
    over what was held; with norms, K is the norm and rotation of the projection of the layer's input."""
    cfg, w, run, prompts, first = setup("fp4", qk_norm)
    seen = [[] for _ in range(cfg.n_layers)]
    for layer, attn in enumerate(run.attn): attn.register_forward_hook(lambda m, args, out, layer=layer: seen[layer].append([t.clone() for t in (*args, out)]))
    n = 40
    run.start_decode(first, use_graph=False)
    before = [[run.caches[l].decompress(s) for s in range(3)] for l in range(cfg.n_layers)]
    run.decode(n)
    for l in range(cfg.n_layers):
        for slot, p in enumerate(prompts):
            k, v = (x.double().cpu() for x in run.caches[l].decompress(slot))
            L = p.shape[0]
            assert k.shape[0] == L + n
            for held, prompt, at in ((k, before[l][slot][0], 1), (v, before[l][slot][1], 2)):
                assert torch.equal(held[:L], prompt.double().cpu())
                assert (held[L:] == R.stored(torch.stack([s[at][slot] for s in seen[l]]))).all()
            for step in (0, 1, 15, 31, n - 1):
                q, _, _, o = seen[l][step]
                ref, tol = R.attention(q[slot], k[:L + step + 1], v[:L + step + 1], run.scale)
                assert ((o[slot].double().cpu() - ref).abs() <= tol).all()
    # layer 0's keys of the first step from its inputs, in 64 bits: the embedding's norm and the projection as torch rounds them, then norm and rotation
    x = torch.nn.functional.rms_norm(w.embed.index_select(0, first), (cfg.hidden,), w.layers[0]["norm1"], cfg.rms_eps)
    qkv = torch.nn.functional.linear(x, w.layers[0]["qkv"]).view(3, -1, 128)
    pos = torch.tensor([p.shape[0] for p in prompts], device=x.device)
    for at, heads, weight in ((0, qkv[:, :8], "q_norm"), (1, qkv[:, 8:10], "k_norm")):
        ref, tol = R.norm_rope(heads, w.layers[0].get(weight), w.cos[pos], w.sin[pos], False, cfg.rms_eps)
        assert ((seen[0][0][at].double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("settings", [dict(temperature=0.9, top_k=50, top_p=0.95), dict(top_p=0.8, min_p=0.01), dict(temperature=0.0)])
@pytest.mark.parametrize("kv", ["fp4", "gaac"])
def test_sampled_steps_in_a_graph_are_the_eager_ones(kv, settings):
    """40 steps replayed and 40 eager ones with the same random numbers: the same tokens, each the definition's choice from that step's logits."""
    n = 40
    u = torch.rand(n, 3, generator=torch.Generator().manual_seed(4)).cuda()
    tokens = []
    for use_graph in (False, True):
        cfg, _, run, prompts, first = setup(kv)
        run.start_decode(first, use_graph=use_graph, sampling=settings)
        out, logits = run.decode(n, keep_logits=True, u=u)
        for i in (0, 7, n - 1):
            for b in range(3):
                want = R.sample(logits[i, b].double().cpu().numpy(), float(u[i, b]), *(float(torch.tensor(settings.get(k, d), dtype=torch.float32)) if k != "top_k" else settings.get(k, 0)
                                for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))))
                assert int(out[i, b]) == want
        tokens.append(out)
        assert run.lens.tolist() == [p.shape[0] + n for p in prompts]
    assert torch.equal(*tokens)
    if settings.get("temperature") == 0.0:      # greedy by sample() and by argmax
        _, _, run, _, first = setup(kv)
        run.start_decode(first)
        assert torch.equal(run.decode(n), tokens[0])


def test_random_numbers_and_sampling_belong_together():
    _, _, run, _, first = setup("fp4")
    run.start_decode(first, use_graph=False, sampling=dict(top_k=5))
    for u in (None, torch.zeros(2, 3, device="cuda"), torch.zeros(3, 2, device="cuda")):
        with pytest.raises(RuntimeError, match=r"decode expects u fp32 \[3, 3\]"): run.decode(3, u=u)
    run.start_decode(first, use_graph=False)
    with pytest.raises(RuntimeError, match="nothing otherwise"): run.decode(3, u=torch.zeros(3, 3, device="cuda"))


def test_a_slot_that_fills_up_is_reported_by_the_loop():
    cfg, w, run, prompts, first = setup("fp4")
    run.start_decode(first)
    run.caches[1].lens[0] = 512      # layer 1 has no room left for row 0
    with pytest.raises(RuntimeError, match="token capacity"): run.decode(16)


def test_caches_from_a_budget_and_their_stats():
    from gaac_amd import FP4KVCache
    from gaac_amd.serving import Attention, DecodeRunner, allocate_fp4_cache, gaac_stats
    cfg, w, run, prompts, first = setup("fp4")
    per_slot = FP4KVCache.bytes_per_slot(cfg.n_kv_heads, cfg.max_len)
    layers = [Attention(8, 128, 0.1, 2) for _ in range(2)]
    with pytest.raises(AssertionError, match="does not fit"): allocate_fp4_cache(layers, 2 * per_slot - 1, 2, cfg.max_len, 4)
    num, caches = allocate_fp4_cache(layers, 5 * per_slot, 2, cfg.max_len, 4)
    assert num == 2 and all(l.fp4 is c and c.n_slots == 2 for l, c in zip(layers, caches))
    assert DecodeRunner(w, n_slots=3, kv="fp4", kv_budget=4 * per_slot).n_slots == 2
    tokens = sum(p.shape[0] for p in prompts)
    st = run.kv_stats()
    assert st["tokens"] == tokens and st["bytes_used"] == tokens * 2 * 136 * 2 and st["bytes_reserved"] == 2 * 3 * per_slot and abs(st["ratio"] - 512 / 136) < 1e-9
    assert gaac_stats(run.caches, 3)["bytes_used"] == st["bytes_used"]
