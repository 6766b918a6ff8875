"""The decode loop on weights in 8 bits, and what its tokens were worth: every operator of prompts and steps against its definition, graphs against eager steps."""
import pytest
import torch

import fp8_ref as R
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def setup(kv, weights="fp8", seed=1, vocab=5000):
    from gaac_amd.serving import DecodeRunner, ModelConfig, Weights
    dev = require_gpu()
    cfg = ModelConfig(hidden=256, n_layers=2, n_heads=8, n_kv_heads=2, ffn=640, vocab=vocab, rope_theta=10000.0, max_len=512, weights=weights)
    w = Weights(cfg, dev, seed=seed)
    g = torch.Generator(device=dev).manual_seed(2)
    prompts = [torch.randint(0, cfg.vocab, (L,), generator=g, device=dev) for L in (200, 37, 64)]
    return cfg, w, DecodeRunner(w, n_slots=3, kv=kv), prompts


def within(a, y, tol):
    a = a.double().cpu()
    assert a.shape == y.shape and ((a - y).abs() <= tol).all()


@pytest.mark.parametrize("kv", ["fp4", "gaac", "bf16"])
def test_every_operator_of_prompts_and_steps(kv, monkeypatch):
    from gaac_amd import FP8Rows, serving
    cfg, w, run, prompts = setup(kv)
    calls = []
    def watch(name):
        f = getattr(serving, name)
        def call(*a, **k):
            out = f(*a, **k)
            calls.append((name, a, k, out))
            return out
        monkeypatch.setattr(serving, name, call)
    for name in ("rms_norm_fp8", "fp8_linear", "fp8_gated"): watch(name)
    first = torch.stack([run.prefill(i, p).argmax() for i, p in enumerate(prompts)])
    run.start_decode(first, use_graph=False)
    run.decode(3)
    passes = 3 + 3
    assert [c[0] for c in calls].count("rms_norm_fp8") == passes * 2 * cfg.n_layers and [c[0] for c in calls].count("fp8_gated") == passes * cfg.n_layers
    assert [c[0] for c in calls].count("fp8_linear") == passes * 3 * cfg.n_layers
    held = lambda x: x.dequantize().double().cpu() if isinstance(x, FP8Rows) else R.stored(x)
    for name, a, k, out in calls:
        if name == "rms_norm_fp8":
            y, h = R.norm(a[0], a[1], a[2], k.get("residual"))
            if k:
                out, got = out
                within(got, h, 2.0 ** -8 * h.abs() * 1.01)
            within(out.dequantize(), y, R.half_step(y) * (1 + 2.0 ** -20) + y.abs() * 2.0 ** -22)
        elif name == "fp8_linear": within(out, *R.product(held(a[0]), a[1].dequantize(), out.dtype))
        else: within(out, *R.gated(held(a[0]), *a[1].dequantize(), out.dtype))
    # the residual goes from one norm into the next
    norms = [c for c in calls if c[0] == "rms_norm_fp8"]
    for i in range(1, 2 * cfg.n_layers):
        before = norms[i - 1][3][1] if norms[i - 1][2] else norms[i - 1][1][0]
        assert torch.equal(norms[i][2]["residual"], before)


@pytest.mark.parametrize("sampling", [None, dict(temperature=0.9, top_k=50)])
@pytest.mark.parametrize("weights", ["fp8", "bf16"])
def test_steps_in_a_graph_and_what_tokens_were_worth(weights, sampling):
    cfg, w, run, prompts = setup("fp4", weights)
    n = 20
    u = None if sampling is None else torch.rand(n, 3, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    out = []
    for graph in (False, True, True):
        first = torch.stack([run.prefill(i, p).argmax() for i, p in enumerate(prompts)])
        run.start_decode(first, use_graph=graph, sampling=sampling, logprobs=4)
        out.append(run.decode(n, keep_logits=True, u=u))
        torch.cuda.synchronize()
    for other in out[1:]:
        assert torch.equal(out[0][0], other[0]) and torch.equal(out[0][1], other[1])
        for a, b in zip(out[0][2], other[2]): assert torch.equal(a, b)
    tokens, logits, worth = out[0]
    assert [tuple(t.shape) for t in worth] == [(n, 3), (n, 3), (n, 3), (n, 3, 4), (n, 3, 4)]
    value, rank, entropy, top_values, top_tokens, tol, tol_entropy = R.logprobs(logits.flatten(0, 1), tokens.flatten(), 4)
    within(worth.logprob.flatten(), value, tol(value))
    within(worth.entropy.flatten(), entropy, tol_entropy)
    within(worth.top_logprobs.flatten(0, 1), top_values, tol(top_values))
    assert torch.equal(worth.rank.flatten().cpu(), rank) and torch.equal(worth.top_tokens.flatten(0, 1).cpu(), top_tokens)
    if sampling is None: assert (worth.rank == 0).all() and torch.equal(worth.top_tokens[..., 0], tokens)
    run.start_decode(first, use_graph=True, sampling=sampling)      # and without
    assert isinstance(run.decode(1, u=None if u is None else u[:1]), torch.Tensor)


@pytest.mark.parametrize("weights", ["fp8", "bf16"])
def test_a_prompt_scored(weights):
    cfg, w, run, prompts = setup("gaac", weights, vocab=20000)
    long = torch.randint(0, cfg.vocab, (400,), generator=torch.Generator().manual_seed(3)).cuda()
    for p in (long, prompts[1], prompts[1][:2], prompts[1][:1]):
        want = run.prefill(0, p)
        logits, worth = run.prefill(0, p, logprobs=3)
        assert torch.equal(logits, want)
        L = len(p)
        assert [tuple(t.shape) for t in worth] == [(L - 1,), (L - 1,), (L - 1,), (L - 1, 3), (L - 1, 3)]
        assert worth.logprob.isfinite().all() and (worth.rank >= 0).all() and (worth.top_logprobs.diff(dim=1) <= 0).all() and (worth.entropy > 0).all()
    # the last token's worth is that of the logits that the prompt without it leaves
    logits, worth = run.prefill(1, long[:257], logprobs=0)
    value, rank, entropy, *_, tol, tol_entropy = R.logprobs(run.prefill(1, long[:256])[None], long[256:257], 0)
    assert abs(worth.logprob[-1].item() - value.item()) < 0.1      # (other sizes, other orders of sums)
    assert run.prefill(1, long[:257], logprobs=0)[1].top_tokens is None


def test_bytes_and_settings():
    from gaac_amd.serving import ModelConfig, Weights
    cfg, w, *_ = setup("bf16")
    _, plain, *_ = setup("bf16", "bf16")
    for a, b in zip(w.layers, plain.layers):
        for name in ("qkv", "o", "down"): assert torch.equal(a[name].dequantize().double().cpu(), R.stored(b[name]))
        for got, want in zip(a["gate_up"].dequantize(), (b["gate_up"][:cfg.ffn], b["gate_up"][cfg.ffn:])): assert torch.equal(got.double().cpu(), R.stored(want))
    projections = sum(t.numel() for l in plain.layers for t in l.values() if t.dim() == 2)
    assert plain.nbytes() - w.nbytes() == 2 * projections - sum(t.nbytes for l in w.layers for t in l.values() if not isinstance(t, torch.Tensor))
    with pytest.raises(RuntimeError, match="bf16 or fp8"): Weights(ModelConfig(hidden=64, n_layers=1, weights="int4"))
    with pytest.raises(RuntimeError, match="no CPU path"): Weights(ModelConfig(hidden=64, n_layers=1, n_heads=2, n_kv_heads=1, ffn=64, vocab=10, weights="fp8"), "cpu")
