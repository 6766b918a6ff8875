"""Numbers of alternatives that cannot be given are refused before a prompt or a step has changed anything."""
import pytest
import torch

from gaac_amd.serving import DecodeRunner, ModelConfig, Weights


@pytest.mark.parametrize("vocab,bad", [(100, 65), (100, -1), (10, 11)])
def test_nothing_is_stored(vocab, bad):
    cfg = ModelConfig(hidden=64, n_layers=1, n_heads=2, n_kv_heads=1, ffn=64, vocab=vocab, max_len=64)
    run = DecodeRunner(Weights(cfg, "cpu"), n_slots=2, kv="bf16")
    tokens = torch.arange(5)
    with pytest.raises(RuntimeError, match=f"prefill gives 0 to {min(64, vocab)} alternatives, not {bad}"): run.prefill(0, tokens, logprobs=bad)
    assert run.lens.tolist() == [0, 0] and not run.caches[0].k.any()
    run.prefill(0, tokens); run.prefill(1, tokens[:3])
    run.start_decode(tokens[:2], use_graph=False)
    before = run.B, run.slots.tolist(), run.dlens.tolist(), run.logprobs
    with pytest.raises(RuntimeError, match=f"start_decode gives 0 to {min(64, vocab)} alternatives, not {bad}"): run.start_decode(tokens[:1], use_graph=False, logprobs=bad)
    assert before == (run.B, run.slots.tolist(), run.dlens.tolist(), run.logprobs) and run.lens.tolist() == [5, 3]
