"""The decode loop's own steps on the CPU, with the model's step in its place taken by a stand-in."""
import pytest
import torch

from gaac_amd import serving
from gaac_amd.serving import DecodeRunner, ModelConfig, Weights

CFG = ModelConfig(hidden=128, n_layers=1, n_heads=2, n_kv_heads=1, ffn=128, vocab=50, max_len=64)


def runner(monkeypatch, logits):
    """A runner whose steps note the tokens that they are given and return `logits` [B, vocab]."""
    run = DecodeRunner(Weights(CFG, "cpu"), n_slots=2, kv="bf16")
    given = []
    def step(tokens, slots, lens, nsplit):
        given.append(tokens.clone())
        lens += 1
        return logits
    monkeypatch.setattr(run, "_step", step)
    return run, given


def test_a_row_without_a_token_goes_on_with_one_that_exists(monkeypatch):
    """sample() returns -1 for a row of nothing but NaN and -inf: the caller sees it, the next step's embedding does not."""
    run, given = runner(monkeypatch, torch.zeros(2, CFG.vocab))
    drawn = iter(([7, -1], [-1, -1], [3, 49]))
    monkeypatch.setattr(serving, "sample", lambda logits, u, **settings: torch.tensor(next(drawn)))
    run.start_decode(torch.tensor([5, 6]), use_graph=False, sampling=dict(top_p=0.9))
    out = run.decode(3, u=torch.zeros(3, 2))
    assert out.tolist() == [[7, -1], [-1, -1], [3, 49]]
    assert [t.tolist() for t in given] == [[5, 6], [7, 0], [0, 0]] and run.tok.tolist() == [3, 49]


def test_likeliest_and_forced_tokens_are_fed_as_they_are(monkeypatch):
    logits = torch.zeros(2, CFG.vocab)
    logits[0, 9] = logits[1, 4] = 1
    run, given = runner(monkeypatch, logits)
    run.start_decode(torch.tensor([5, 6]), use_graph=False)
    assert run.decode(2).tolist() == [[9, 4], [9, 4]] and [t.tolist() for t in given] == [[5, 6], [9, 4]]
    assert run.decode(2, forced=torch.tensor([[1, 2], [3, 8]])).tolist() == [[9, 4], [9, 4]] and [t.tolist() for t in given[2:]] == [[9, 4], [1, 2]]
    assert run.tok.tolist() == [3, 8]


def test_rows_do_not_grow_past_the_models_positions(monkeypatch):
    """Refused before anything runs: a step behind the last position would be one of NaN, over tokens that the caches left out."""
    run, given = runner(monkeypatch, torch.zeros(2, CFG.vocab))
    run.lens.copy_(torch.tensor([10, 60]))
    run.start_decode(torch.tensor([5, 6]), use_graph=False)
    with pytest.raises(RuntimeError, match="decode of 5 steps: the longest row holds 60 tokens, the model's positions end at 64"): run.decode(5)
    assert not given and run.lens.tolist() == [10, 60]
    run.decode(3)
    with pytest.raises(RuntimeError, match="holds 63 tokens"): run.decode(2)
    run.decode(1)
    assert run.lens.tolist() == [14, 64] and len(given) == 4
    with pytest.raises(RuntimeError, match="holds 64 tokens"): run.decode(1)
    run.dlens.copy_(torch.tensor([14, 20]))      # tokens taken back
    run.decode(40)
    assert run.lens.tolist() == [54, 60]
    with pytest.raises(RuntimeError, match="prompt has 65 tokens"): run.prefill(0, torch.zeros(65, dtype=torch.int64))
