"""What a prompt's tokens were worth, bit for bit: each score is of the token behind a position, from that position's own logits."""
import pytest
import torch

from gpu_util import require_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", ["fp8", "bf16"])
@pytest.mark.parametrize("L", [2, 700, 1024, 1025, 1026, 2500])
def test_scores_are_those_of_their_positions(L, weights, monkeypatch):
    from gaac_amd import token_logprobs
    from gaac_amd.serving import DecodeRunner, ModelConfig, Weights
    dev = require_gpu()
    cfg = ModelConfig(hidden=256, n_layers=2, n_heads=8, n_kv_heads=2, ffn=640, vocab=20000, rope_theta=10000.0, max_len=3000, weights=weights)
    run = DecodeRunner(Weights(cfg, dev, seed=1), n_slots=1, kv="gaac")
    tokens = torch.randint(0, cfg.vocab, (L,), generator=torch.Generator().manual_seed(L)).cuda()
    seen = []
    layers = run._layers
    monkeypatch.setattr(run, "_layers", lambda x, pos: seen.append(layers(x, pos)) or seen[-1])
    last, worth = run.prefill(0, tokens, logprobs=5)
    x, = seen
    assert x.shape == (L, cfg.hidden) and all(len(t) == L - 1 for t in worth)
    # positions 0 .. L - 2, the logits made by the same calls, of 1024 positions each
    for i in range(0, L - 1, 1024):
        n = min(1024, L - 1 - i)
        want = token_logprobs(run._logits(x[i:i + n]), tokens[i + 1:i + 1 + n], top=5)
        for a, b in zip(worth, want): assert torch.equal(a[i:i + n], b)
    # a position's score depends on its own row and on no other: the same rows by themselves and in another order
    at = torch.randperm(L - 1, generator=torch.Generator().manual_seed(1)).cuda()[:1024]
    logits = run._logits(x[:-1][:1024])
    at = at[at < len(logits)]
    want = token_logprobs(logits[at], tokens[at + 1], top=5)
    for a, b in zip(worth, want): assert torch.equal(a[at], b)
    # and neighbours have others (the test can tell)
    if L > 100:
        shifted = token_logprobs(logits[1:], tokens[1:len(logits)], top=5)
        assert (shifted.logprob != worth.logprob[:len(logits) - 1]).float().mean() > 0.99
    assert torch.equal(last, run._logits(x[-1:])[0].float())
