"""The decode loop at its limits: rows without a token, rows that are full."""
import pytest
import torch

from gpu_util import require_gpu

pytestmark = pytest.mark.gpu


def setup(kv, n_slots=3, max_len=512, lens=(200, 37, 64)):
    from gaac_amd.serving import DecodeRunner, ModelConfig, Weights
    dev = require_gpu()
    cfg = ModelConfig(hidden=256, n_layers=2, n_heads=8, n_kv_heads=2, ffn=512, vocab=5000, rope_theta=10000.0, max_len=max_len)
    w = Weights(cfg, dev, seed=1)
    run = DecodeRunner(w, n_slots=n_slots, kv=kv)
    g = torch.Generator(device=dev).manual_seed(2)
    first = torch.stack([run.prefill(i, torch.randint(0, cfg.vocab, (L,), generator=g, device=dev)).argmax() for i, L in enumerate(lens)])
    return cfg, w, run, first


@pytest.mark.parametrize("kv", ["fp4", "gaac", "bf16"])
@pytest.mark.parametrize("use_graph", [False, True])
def test_rows_without_a_token(kv, use_graph):
    """A model whose logits are all NaN: every drawn token is -1, and no step is given it."""
    cfg, w, run, first = setup(kv)
    w.final_norm.fill_(float("nan"))
    run.start_decode(first, use_graph=use_graph, sampling=dict(top_k=50, top_p=0.9))
    out = run.decode(4, u=torch.full((4, 3), 0.5, device="cuda"))
    assert (out == -1).all() and run.tok.tolist() == [0, 0, 0]
    w.final_norm.fill_(1.0)
    out = run.decode(4, u=torch.full((4, 3), 0.5, device="cuda"))
    assert ((out >= 0) & (out < cfg.vocab)).all() and torch.equal(out[-1], run.tok)


@pytest.mark.parametrize("kv", ["fp4", "gaac", "bf16"])
@pytest.mark.parametrize("use_graph", [False, True])
def test_rows_up_to_the_last_position(kv, use_graph):
    """max_len is no whole number of tiles: the last steps that fit are finite, one more is refused and leaves everything as it was."""
    cfg, w, run, first = setup(kv, max_len=75, lens=(70, 37, 64))
    settings = dict(temperature=0.8, top_k=20)
    run.start_decode(first, use_graph=use_graph, sampling=settings)
    u = torch.full((6, 3), 0.5, device="cuda")
    with pytest.raises(RuntimeError, match="the longest row holds 70 tokens, the model's positions end at 75"): run.decode(6, u=u)
    out, logits = run.decode(5, keep_logits=True, u=u[:5])
    assert (out >= 0).all() and logits.isfinite().all() and run.lens.tolist() == [75, 42, 69]
    with pytest.raises(RuntimeError, match="holds 75 tokens"): run.decode(1, u=u[:1])
    assert run.lens.tolist() == [75, 42, 69]
    if kv != "bf16":
        for c in run.caches: assert c.decompress(0)[0].shape[0] == 75
