"""The operators of a model with 8-bit weights, and of the log probabilities of what it says, as timed cases: through the package's entry points (own = True) or in plain torch operations.

Four kinds of work, in the order a step meets them:

  norm       the residual's addition and the root-mean-square norm, its result in 8 bits, read back                       rms_norm_fp8, FP8Rows.dequantize
  linear     rows of activations by a weight in 8 bits                                                                    fp8_linear
  ffn        a gated feed-forward block: both projections, silu and product, the way back                                 fp8_gated, fp8_linear
  logprobs   log probabilities of given tokens, their ranks, the entropy, the likeliest alternatives                      token_logprobs

8 bits: 128 consecutive elements of a row share a power of two 2^E, the smallest with max |x| <= 448 * 2^E, from -117 to 119, and an element is the nearest e4m3 number (ties to the even
code) times 2^E; weights the same way along their inputs.  Activations are quantised from the type they come in, in every product; the gated block's inner result is rounded to bf16 first, as its output is.

Activations are Gaussian with channel scales log-uniform in 2^[-2, 2] and one channel in 200 sixteen times larger, as a trained model's; weights are Gaussian of
standard deviation 1/sqrt(K).  Logits are a wide Gaussian with a few dozen likely tokens above it."""
import math

import torch

own = False

BLOCK = 128             # elements of a row that share a power of two

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the decode step of four sequences, a model of width 4096: launches are everything
        dict(name="norm_step_4", kind="norm", M=4, K=4096, dtype="bf16", residual=True),
        # a prompt of odd length, a width that ends inside a block, the first norm of a model (no residual yet)
        dict(name="norm_777_odd", kind="norm", M=777, K=5000, dtype="fp16", residual=False),
        # a long prompt
        dict(name="norm_16k", kind="norm", M=16384, K=4096, dtype="bf16", residual=True),
        # the decode step of four sequences: queries, keys and values of 32 + 2 * 8 heads
        dict(name="linear_step_4", kind="linear", M=4, K=4096, N=6144, dtype="bf16"),
        # a busy server's decode step: the way back from the inner width
        dict(name="linear_48", kind="linear", M=48, K=14336, N=4096, dtype="bf16"),
        # a few short prompts together: the heads' outputs
        dict(name="linear_200", kind="linear", M=200, K=4096, N=4096, dtype="fp32"),
        # a prompt of odd length
        dict(name="linear_777", kind="linear", M=777, K=4096, N=6144, dtype="fp16"),
        # a long prompt, the widest product of the model
        dict(name="linear_8k", kind="linear", M=8192, K=4096, N=28672, dtype="bf16"),
        # the decode step of four sequences
        dict(name="ffn_step_4", kind="ffn", M=4, K=4096, F=14336, dtype="bf16"),
        # a prompt of ordinary length
        dict(name="ffn_2k", kind="ffn", M=2048, K=4096, F=14336, dtype="bf16"),
        # the end of a decode step: what the step's tokens were worth, and twenty alternatives each
        dict(name="logprobs_4", kind="logprobs", B=4, V=128256, dtype="bf16", top=20),
        # a prompt of odd length scored
        dict(name="logprobs_777", kind="logprobs", B=777, V=128256, dtype="fp32", top=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: most are whole blocks, some whole groups of 16, some anything."""
    n, step = _log(rng, lo, hi), rng.choice([128, 128, 128, 16, 1])
    return max(step, n // step * step)


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "linear", "ffn", "ffn", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "norm":
        K = _width(rng, 64, 16384)
        return dict(kind=kind, M=min(_log(rng, 1, 16384), (48 << 20) // K), K=K, dtype=dtype, residual=rng.random() < 0.7)
    if kind == "linear":
        K, N = _width(rng, 128, 16384), _width(rng, 64, 28672)
        return dict(kind=kind, M=min(_log(rng, 1, 8192), (1 << 38) // (K * N)), K=K, N=N, dtype=dtype)
    if kind == "ffn":
        K, F = _width(rng, 256, 8192), _width(rng, 512, 14336)
        return dict(kind=kind, M=min(_log(rng, 1, 4096), (1 << 36) // (K * F)), K=K, F=F, dtype=dtype)
    V = _log(rng, 1000, 262144)
    return dict(kind=kind, B=min(_log(rng, 1, 1024), 64000000 // V), V=V, dtype=dtype, top=rng.choice([0, 1, 5, 20, 64]))


# ---------------------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """What comes in, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    uniform = lambda *shape: torch.rand(*shape, generator=g, device="cuda")
    t = TYPES[case["dtype"]]
    if case["kind"] == "logprobs":
        B, V = case["B"], case["V"]
        x = normal(B, V).mul_(2.5)
        at = torch.randint(0, V, (B, 48), generator=g, device="cuda")
        x.scatter_add_(1, at, uniform(B, 48) * 10 + 2)
        x[:, torch.randint(0, V, (V // 50,), generator=g, device="cuda")] = -math.inf      # tokens that may not come
        tokens = torch.where(uniform(B) < 0.7, at[:, 0], torch.randint(0, V, (B,), generator=g, device="cuda"))
        return dict(logits=x.to(t), tokens=tokens)
    M, K = case["M"], case["K"]
    channels = torch.exp2(uniform(K) * 4 - 2) * torch.where(uniform(K) < 0.005, 16.0, 1.0)
    out = dict(x=normal(M, K).mul_(channels).to(t))
    weight = lambda n, k: normal(n, k).mul_(k ** -0.5).to(torch.bfloat16)
    if case["kind"] == "norm":
        out.update(weight=(uniform(K) + 0.5).to(t), residual=normal(M, K).mul_(channels).mul_(4).to(t) if case["residual"] else None)
    elif case["kind"] == "linear":
        out.update(weights=[(weight(case["N"], K),)])
    else:
        out.update(weights=[(weight(case["F"], K), weight(case["F"], K)), (weight(K, case["F"]),)])
    return out


# ---------------------------------------------------------------------------------------------------- plain forms
def _quantise(x):
    """x fp32 [M, K] -> e4m3 [M, blocks, 128] (zeros behind K) and exponents int32 [M, blocks]."""
    M, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % BLOCK)).view(M, -1, BLOCK)
    E = (((b.abs().amax(-1).view(torch.int32) + 0x1FFFFF) >> 23) - 135).clamp(min=-117, max=119)
    return (b * ((127 - E) << 23).view(torch.float32).unsqueeze(-1)).to(torch.float8_e4m3fn), E


def _values(codes, E):
    """The fp32 [M, blocks * 128] values that codes and exponents stand for."""
    return (codes.float() * ((E + 127) << 23).view(torch.float32).unsqueeze(-1)).flatten(1)


def _product(x, weight):
    """x fp32 [M, K] in 8 bits by a weight (codes and exponents): fp32 [M, N]."""
    return torch.matmul(_values(*_quantise(x)), _values(*weight).T)


def _plain_logprobs(logits, tokens, top):
    x = logits.float()
    at = tokens[:, None]
    shifted = x - x.amax(-1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(-1)
    lse = torch.log(total)
    mine = x.gather(1, at)
    index = torch.arange(x.shape[1], device=x.device)
    rank = ((x > mine) | ((x == mine) & (index < at))).sum(-1)
    entropy = lse - torch.where(e > 0, e * shifted, 0.0).sum(-1) / total
    out = [shifted.gather(1, at)[:, 0] - lse, rank, entropy]
    if top:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
        out += [shifted.gather(1, order) - lse[:, None], order]
    return out


# ---------------------------------------------------------------------------------------------------- the cases
def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if "weights" in s:      # laid out once, as a program keeps them
        if own:
            from gaac_amd import FP8Weight
            s["weights"] = [FP8Weight(*w) for w in s["weights"]]
        else:
            s["weights"] = [[_quantise(part.float()) for part in w] for w in s["weights"]]
    return s


def run(s):
    case = s["case"]
    kind, t = case["kind"], TYPES[case["dtype"]]
    if own:
        import gaac_amd
        if kind == "norm":
            if s["residual"] is None:
                return [gaac_amd.rms_norm_fp8(s["x"], s["weight"], 1e-5).dequantize()]
            rows, h = gaac_amd.rms_norm_fp8(s["x"], s["weight"], 1e-5, residual=s["residual"])
            return [rows.dequantize(), h]
        if kind == "linear":
            return gaac_amd.fp8_linear(s["x"], s["weights"][0])
        if kind == "ffn":
            return gaac_amd.fp8_linear(gaac_amd.fp8_gated(s["x"], s["weights"][0]), s["weights"][1], out_dtype=torch.bfloat16)
        return [x for x in gaac_amd.token_logprobs(s["logits"], s["tokens"], top=case["top"]) if x is not None]
    if kind == "norm":
        h = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * s["weight"].float()
        values = _values(*_quantise(y))[:, :case["K"]].to(torch.bfloat16)
        return [values] if s["residual"] is None else [values, h.to(t)]
    if kind == "linear":
        return _product(s["x"].float(), s["weights"][0][0]).to(t)
    if kind == "ffn":
        (gate, up), (down,) = s["weights"]
        g, u = _product(s["x"].float(), gate), _product(s["x"].float(), up)
        return _product((g / (1 + torch.exp(-g)) * u).to(torch.bfloat16).float(), down).to(torch.bfloat16)
    return _plain_logprobs(s["logits"], s["tokens"], case["top"])


def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "logprobs":
        return dict(bytes=case["B"] * (case["V"] * size + 24 + 12 * case["top"]), flops=0)
    M, K = case["M"], case["K"]
    if kind == "norm":      # rows in (and the residual in and out), 8 bits out, in again, their values out
        return dict(bytes=M * K * ((3 if case["residual"] else 1) * size + 1 + 1 + 2) + K * size, flops=0)
    if kind == "linear":
        return dict(bytes=M * K * size + case["N"] * K + M * case["N"] * size, flops=2 * M * K * case["N"])
    return dict(bytes=M * K * (size + 2) + 3 * case["F"] * K, flops=6 * M * K * case["F"])


# ---------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _stored64(x):
    """What 8 bits hold of x, by the definition."""
    x = x.double()
    M, K = x.shape
    b = torch.cat([x, x.new_zeros(M, -K % BLOCK)], 1).view(M, -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    E = torch.floor(torch.log2(top.clamp(min=1e-300))) - 10      # below the smallest power that will do
    for _ in range(4):
        E = torch.where(top > 448 * torch.exp2(E), E + 1, E)
    s = torch.exp2(E.clamp(min=-117, max=119))
    y = b / s
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step * s).flatten(1)[:, :K]


def _rounded64(x):
    """x in 64 bits rounded to bf16's 8 bits of mantissa."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=1e-30))) - 7)
    return torch.round(x / step) * step


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "norm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["K"] + 1e-5) * s["weight"].double()
        return [_stored64(y)] if s["residual"] is None else [_stored64(y), h]
    if kind == "logprobs":
        value, rank, entropy, alternatives, order = [], [], [], [], []
        index = torch.arange(case["V"], device="cuda")
        for row, token in zip(s["logits"], s["tokens"]):
            row = row.double()
            p = torch.log_softmax(row, 0)
            value.append(p[token])
            rank.append((row > row[token]).sum() + ((row == row[token]) & (index < token)).sum())
            entropy.append(-(p.exp() * p.clamp(min=-1e300)).sum())
            if case["top"]:
                order.append(torch.sort(row, descending=True, stable=True).indices[:case["top"]])
                alternatives.append(p[order[-1]])
        return [torch.stack(x) for x in (value, rank, entropy, alternatives, order) if x]
    x = _stored64(s["x"])
    if kind == "linear":
        return x @ _stored64(s["weights"][0][0]).T.contiguous()
    (gate, up), (down,) = s["weights"]
    g, u = x @ _stored64(gate).T.contiguous(), x @ _stored64(up).T.contiguous()
    return _stored64(_rounded64(g * torch.sigmoid(g) * u)) @ _stored64(down).T.contiguous()
