"""The operators of a decode step on a 4-bit cache, as timed cases: through the package's entry points (own = True) or in plain torch operations.

Five kinds of work, in the order a step meets them:

  rope       norms of queries and keys for each head and their rotation, on views of the fused projection's output       qk_norm_rope
  prompt     a prompt into a slot of the 4-bit cache, and all of it read back                                              FP4KVCache.prefill / decompress
  request    a short request on one layer: prompts into slots, then decode steps                                           FP4KVCache.prefill / append / attention
  attend     one decode step's attention of a batch over the 4-bit cache                                                   FP4KVCache.attention
  sample     one token per row from its logits: temperature, top-k, top-p, min-p, with given random numbers                sample

The cache holds MXFP4: 32 consecutive channels of one token and head share a power of two 2^E, the smallest with max |x| < 7 * 2^E, from -125 to 125,
and an element is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^E (ties to the even code; 6 beyond it), with its sign; a block that is not finite reads as NaN.

K and V are Gaussian per (kv head, channel) with channel scales log-uniform in 2^[-2, 2], and queries are standard normal: a softmax that spreads over many
tokens.  Logits are a wide Gaussian with a few dozen likely tokens above it, as a trained model's."""
import math

import numpy as np
import torch

own = False

D = 128
BLOCK = 32              # channels that share a power of two
ROW = D // 2 + D // BLOCK      # bytes of one (token, kv head) row of K or of V in the cache
RAW = 2 * D             # the same row in bf16

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the decode step of four sequences, 32 query / 8 kv heads: launches are everything
        dict(name="rope_step_4", kind="rope", N=4, n_q=32, n_kv=8, D=128, R=128, dtype="bf16", norm=True, interleaved=False, max_pos=33024),
        # a prompt of odd length in one pass, 24 query / 4 kv heads, half of each head rotated, in pairs of neighbours
        dict(name="rope_777_partial", kind="rope", N=777, n_q=24, n_kv=4, D=128, R=64, dtype="fp16", norm=True, interleaved=True, max_pos=4096),
        # a long prompt, 32 query / 8 kv heads
        dict(name="rope_16k", kind="rope", N=16384, n_q=32, n_kv=8, D=128, R=128, dtype="bf16", norm=True, interleaved=False, max_pos=33024),
        # a chat turn's prompt, of a length that ends inside a tile
        dict(name="prompt_777", kind="prompt", n_kv=8, L=777),
        # a long prompt
        dict(name="prompt_32k", kind="prompt", n_kv=8, L=32768),
        # four short requests on one layer: prompts, then sixteen decode steps
        dict(name="request_333", kind="request", B=4, n_kv=8, G=4, L=333, steps=16),
        # a chat turn with a short context: launches and latency are everything
        dict(name="attend_1k", kind="attend", B=1, n_kv=8, G=4, lo=1000, hi=1000),
        # the long-context decode step: one sequence, 32 query / 8 kv heads, 64K tokens
        dict(name="attend_64k", kind="attend", B=1, n_kv=8, G=4, lo=65536, hi=65536),
        # one layer of a busy chat server: many ragged short sequences
        dict(name="attend_32_chat", kind="attend", B=32, n_kv=8, G=4, lo=300, hi=6000),
        # one layer of a serving step: 16 sequences of very different lengths up to 64K
        dict(name="attend_16x64k", kind="attend", B=16, n_kv=8, G=4, lo=4096, hi=65536),
        # the end of a decode step of four sequences over a vocabulary of 128256
        dict(name="sample_4", kind="sample", B=4, V=128256, dtype="bf16", temperature=0.7, top_k=50, top_p=0.95, min_p=0.0, mixed=False),
        # a busy server: every row with settings of its own, some greedy, logits in 32 bits
        dict(name="sample_64_mixed", kind="sample", B=64, V=128256, dtype="fp32", temperature=1.0, top_k=0, top_p=0.9, min_p=0.02, mixed=True),
    ]


HEADS = [(8, 4), (8, 4), (4, 6), (8, 2), (4, 8), (2, 8), (8, 1), (1, 16), (8, 5), (16, 2)]      # (kv heads, query heads per kv head)
MOST_ROWS = 4 << 20      # (token, kv head) rows of a drawn batch: below the listed serving step's


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "prompt", "request", "attend", "attend", "sample", "sample"])
    n_kv, G = rng.choice(HEADS)
    if kind == "rope":
        d = rng.choice([64, 128, 128, 256])
        return dict(kind=kind, N=_log(rng, 1, 8192), n_q=n_kv * G, n_kv=n_kv, D=d, R=rng.choice([d, d, d // 2, d // 4]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    norm=rng.random() < 0.7, interleaved=rng.random() < 0.3, max_pos=_log(rng, 100, 131072))
    if kind == "prompt":
        return dict(kind=kind, n_kv=n_kv, L=_log(rng, 1, 32768))
    if kind == "request":
        return dict(kind=kind, B=rng.randint(1, 4), n_kv=n_kv, G=G, L=_log(rng, 1, 1000), steps=rng.randint(8, 16))
    if kind == "attend":
        B = _log(rng, 1, 48)
        hi = min(_log(rng, 20, 65536), MOST_ROWS // (B * n_kv))
        return dict(kind=kind, B=B, n_kv=n_kv, G=G, lo=_log(rng, 1, hi), hi=hi)
    V = _log(rng, 1000, 262144)
    return dict(kind=kind, B=min(_log(rng, 1, 256), 8000000 // V), V=V, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]),
                top_k=rng.choice([0, 0, 1, 20, 50, 300]), top_p=rng.choice([1.0, 0.5, 0.9, 0.95, 0.999]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), mixed=rng.random() < 0.3)


def _lengths(case):
    """B lengths spread evenly from lo to hi, in an order that is not sorted."""
    n = case["B"]
    lens = [case["lo"] + (case["hi"] - case["lo"]) * (2 * i + 1) // (2 * n) for i in range(n)] if n > 1 else [case["hi"]]
    return [lens[(5 * i + 2) % n] for i in range(n)] if n % 5 else [lens[(7 * i + 2) % n] for i in range(n)] if n % 7 else lens


# ---------------------------------------------------------------------------------------------------- inputs
class _Rows:
    """K or V rows [n, n_kv, D] bf16 with fixed channel scales."""
    def __init__(self, g, n_kv):
        self.g, self.n_kv = g, n_kv
        self.sigma = torch.exp2(torch.rand(1, n_kv, D, generator=g, device="cuda") * 4 - 2)

    def __call__(self, n):
        return torch.randn(n, self.n_kv, D, generator=self.g, device="cuda").mul_(self.sigma).to(torch.bfloat16)


def _query(g, B, n_q):
    return torch.randn(B, n_q, D, generator=g, device="cuda").to(torch.bfloat16)


def _inputs(case, seed):
    """What comes in, from the seed alone.  Of a batch's contexts a function that makes them one after the other."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]
    if kind == "rope":
        t, n_kv, d = TYPES[case["dtype"]], case["n_kv"], case["D"]
        heads = case["n_q"] + 2 * n_kv
        qkv = (torch.randn(case["N"], heads, d, generator=g, device="cuda") * torch.exp2(torch.rand(1, heads, d, generator=g, device="cuda") * 4 - 2)).to(t)
        w = [(torch.rand(d, generator=g, device="cuda") + 0.5).to(t) for _ in range(2)] if case["norm"] else [None, None]
        pos = torch.randint(0, case["max_pos"], (case["N"],), generator=g, device="cuda")
        freq = 500000.0 ** -(torch.arange(0, case["R"], 2, device="cuda", dtype=torch.float64) / case["R"])
        ang = torch.arange(case["max_pos"], device="cuda", dtype=torch.float64)[:, None] * freq
        return dict(q=qkv[:, :case["n_q"]], k=qkv[:, case["n_q"]:case["n_q"] + n_kv], w=w, pos=pos, cos=ang.cos().float(), sin=ang.sin().float())
    if kind == "sample":
        B, V = case["B"], case["V"]
        x = torch.randn(B, V, generator=g, device="cuda") * 2.5
        at = torch.randint(0, V, (B, 48), generator=g, device="cuda")
        x.scatter_add_(1, at, torch.rand(B, 48, generator=g, device="cuda") * 10 + 2)
        x.masked_fill_(torch.rand(B, V, generator=g, device="cuda") < 0.02, -math.inf)      # tokens that may not come
        out = dict(logits=x.to(TYPES[case["dtype"]]), u=torch.rand(B, generator=g, device="cuda"))
        rows = dict(temperature=torch.full((B,), case["temperature"]), top_k=torch.full((B,), case["top_k"], dtype=torch.int32),
                    top_p=torch.full((B,), case["top_p"]), min_p=torch.full((B,), case["min_p"]))
        if case["mixed"]:      # settings of every kind side by side
            i = torch.arange(B)
            rows["temperature"] = torch.where(i % 7 == 3, 0.0, rows["temperature"] * (0.5 + 0.25 * (i % 4)))
            rows["top_k"] = torch.where(i % 3 == 1, 40, rows["top_k"]).int()
            rows["top_p"] = torch.where(i % 5 == 2, 1.0, rows["top_p"])
            rows["min_p"] = torch.where(i % 2 == 1, 0.0, rows["min_p"])
        out["rows"] = {k: v.to("cuda") for k, v in rows.items()}
        return out
    n_kv = case["n_kv"]
    kr, vr = _Rows(g, n_kv), _Rows(g, n_kv)
    if kind == "prompt":
        return dict(k=kr(case["L"]), v=vr(case["L"]))
    n_q = n_kv * case["G"]
    if kind == "request":
        B = case["B"]
        prompts = [(kr(case["L"]), vr(case["L"])) for _ in range(B)]
        return dict(prompts=prompts, new=[(_query(g, B, n_q), kr(B), vr(B)) for _ in range(case["steps"])])
    q = _query(g, case["B"], n_q)      # row b reads slot B - 1 - b
    return dict(q=q, contexts=lambda: ((i, kr(L), vr(L)) for i, L in enumerate(_lengths(case))))


# ---------------------------------------------------------------------------------------------------- plain forms
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x):
    """x [..., D] -> codes uint8 [..., D/2] (an even channel in the low half of its byte), exponent bytes uint8 [..., D/32]."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1)
    E = (((top.view(torch.int32) + 0x200000) >> 23) - 129).clamp(min=-125, max=125)
    y = b.abs() * ((127 - E) << 23).view(torch.float32).unsqueeze(-1)
    code = (y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0) + 8 * (b < 0)
    code = code.to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.where(torch.isfinite(top), E + 127, 255).to(torch.uint8)


def _values(codes, exps):
    """The fp32 [..., D] values that codes and exponent bytes stand for."""
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device=codes.device)
    v = grid[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    s = torch.where(exps == 255, math.nan, (exps.int() << 23).view(torch.float32))
    return (v.unflatten(-1, (-1, BLOCK)) * s.unsqueeze(-1)).flatten(-2)


class _PlainCache:
    """Token rows of every slot, [capacity, n_kv, .] each."""
    def __init__(self, n_slots, n_kv, capacity):
        new = lambda *shape: torch.zeros(n_slots, capacity, n_kv, *shape, dtype=torch.uint8, device="cuda")
        self.n_kv, self.codes, self.exps = n_kv, (new(D // 2), new(D // 2)), (new(D // BLOCK), new(D // BLOCK))
        self.lens = [0] * n_slots

    def put(self, slot, at, k, v):
        for i, x in enumerate((k, v)):
            c, e = _quantise(x)
            self.codes[i][slot, at:at + len(x)] = c
            self.exps[i][slot, at:at + len(x)] = e
        self.lens[slot] = at + len(k)

    def rows(self, slot):
        return [_values(self.codes[i][slot, :self.lens[slot]], self.exps[i][slot, :self.lens[slot]]) for i in range(2)]

    def attention(self, q, slots):
        return torch.stack([_attend(q[b].float(), *self.rows(s), D ** -0.5) for b, s in enumerate(slots)]).to(torch.bfloat16)


def _attend(q, k, v, scale):
    """q [n_q, D], k, v [L, n_kv, D], all of one type: softmax(scale q k^T) v."""
    n_kv = k.shape[1]
    s = torch.matmul(q.view(n_kv, -1, D), k.permute(1, 2, 0).contiguous()) * scale
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (torch.matmul(p, v.transpose(0, 1).contiguous()) / p.sum(-1, keepdim=True)).view(-1, D)


def _norm_rope(x, w, cos, sin, interleaved, eps):
    """x [N, heads, D] in the type to compute in, cos, sin [N, R/2]."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    half = cos.shape[-1]
    c, s, rot, rest = cos[:, None], sin[:, None], x[..., :2 * half], x[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    a, b = a * c - b * s, b * c + a * s
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), rest], -1)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    x = logits.double()
    B, V = x.shape
    top = x.amax(-1, keepdim=True)
    greedy = temperature <= 0
    T = torch.where(greedy, 1.0, temperature.double())[:, None]
    w = torch.exp((x - top) / T)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(V, device=x.device)
    ws = torch.where((top_k[:, None] <= 0) | (rank < top_k[:, None]), ws, 0.0)
    run = ws.cumsum(-1)
    before = torch.cat([torch.zeros_like(run[:, :1]), run[:, :-1]], -1)
    p = top_p.double()[:, None]
    ws = torch.where((p >= 1) | (before < p * run[:, -1:]) | (rank == 0), ws, 0.0)
    ws = torch.where(ws >= min_p.double()[:, None], ws, 0.0)
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    run = kept.cumsum(-1)
    token = (run <= u.double()[:, None] * run[:, -1:]).sum(-1)
    first = torch.where(x == top, rank, V).amin(-1)
    return torch.where(greedy, first, token)


# ---------------------------------------------------------------------------------------------------- the cases
def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    kind = case["kind"]
    if kind in ("rope", "sample"):
        if kind == "sample" and own and not case["mixed"]:      # one setting for all rows
            s["rows"] = {k: case[k] for k in s["rows"]}
        return s
    B = case.get("B", 1)
    n_kv, room = case["n_kv"], {"prompt": lambda: case["L"], "request": lambda: case["L"] + case["steps"], "attend": lambda: case["hi"]}[kind]()
    if own:
        from gaac_amd import FP4KVCache
        s["cache"] = FP4KVCache(B, n_kv, room)
    else:
        s["cache"] = _PlainCache(B, n_kv, room)
    order = list(range(B)) if kind == "request" else list(range(B - 1, -1, -1))
    s["slots"] = torch.tensor(order, dtype=torch.int32, device="cuda") if own else order
    if kind == "attend":
        for i, k, v in s.pop("contexts")():
            s["cache"].prefill(i, k, v) if own else s["cache"].put(i, 0, k, v)
    return s


def run(s):
    case, cache = s["case"], s.get("cache")
    kind = case["kind"]
    if kind == "rope":
        if own:
            from gaac_amd import qk_norm_rope
            return qk_norm_rope(s["q"], s["k"], s["pos"], s["cos"], s["sin"], *s["w"], eps=1e-6, interleaved=case["interleaved"])
        cos, sin = s["cos"][s["pos"]], s["sin"][s["pos"]]
        return tuple(_norm_rope(x.float(), w if w is None else w.float(), cos, sin, case["interleaved"], 1e-6).to(x.dtype) for x, w in zip((s["q"], s["k"]), s["w"]))
    if kind == "sample":
        if own:
            from gaac_amd import sample
            return sample(s["logits"], s["u"], **s["rows"])
        return _plain_sample(s["logits"], s["u"], **s["rows"])
    if kind == "prompt":
        if own:
            cache.prefill(0, s["k"], s["v"])
            return cache.decompress(0)
        cache.put(0, 0, s["k"], s["v"])
        return tuple(x.to(torch.bfloat16) for x in cache.rows(0))
    if kind == "attend":
        return cache.attention(s["q"], s["slots"], D ** -0.5, max_len=case["hi"]) if own else cache.attention(s["q"], s["slots"])
    out = []
    for i, (k, v) in enumerate(s["prompts"]):
        cache.prefill(i, k, v) if own else cache.put(i, 0, k, v)
    for step, (q, k, v) in enumerate(s["new"]):
        if own:
            cache.append(s["slots"], k, v)
            out.append(cache.attention(q, s["slots"], D ** -0.5))
        else:
            for b in s["slots"]:
                cache.put(b, case["L"] + step, k[b:b + 1], v[b:b + 1])
            out.append(cache.attention(q, s["slots"]))
    return out


def work(case):
    kind = case["kind"]
    if kind == "rope":      # heads in and out, a row of cos and of sin a token, the positions
        return dict(bytes=case["N"] * (2 * (case["n_q"] + case["n_kv"]) * case["D"] * SIZE[case["dtype"]] + 4 * case["R"] + 8), flops=6 * case["N"] * (case["n_q"] + case["n_kv"]) * case["D"])
    if kind == "sample":
        return dict(bytes=case["B"] * (case["V"] * SIZE[case["dtype"]] + 12), flops=0)
    n_kv = case["n_kv"]
    if kind == "prompt":      # rows in, into the cache, out of it, values out
        return dict(bytes=2 * n_kv * case["L"] * (RAW + ROW + ROW + RAW), flops=0)
    G, B = case["G"], case["B"]
    qo = 2 * n_kv * G * RAW      # one row's queries in and outputs out
    if kind == "attend":
        rows, stored = sum(_lengths(case)), 0
    else:
        rows, stored = sum(B * (case["L"] + i + 1) for i in range(case["steps"])), B * (case["L"] + case["steps"])
        B *= case["steps"]
    return dict(bytes=2 * n_kv * (rows * ROW + stored * (RAW + ROW)) + B * qo, flops=4 * n_kv * G * D * rows)


# ---------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _stored64(x):
    """What the cache holds of x, by the definition: the nearest grid value of each element, found by distance."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    E = torch.floor(torch.log2(top.clamp(min=1e-300))) - 3      # at or below the smallest power that will do
    for _ in range(4):
        E = torch.where(top >= 7 * torch.exp2(E), E + 1, E)
    s = torch.exp2(E.clamp(min=-125, max=125))
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    y = b.abs() / s
    best, value = torch.full_like(y, math.inf), torch.zeros_like(y)
    for i in (0, 2, 4, 6, 1, 3, 5, 7):      # even codes first: a tie stays with them
        d = (y - grid[i]).abs()
        nearer = d < best
        best, value = torch.where(nearer, d, best), torch.where(nearer, grid[i], value)
    return (value * s * torch.where(b < 0, -1.0, 1.0)).flatten(-2)


def _attend64(q, k, v):
    out = []
    n_kv, G = k.shape[1], q.shape[0] // k.shape[1]
    for h in range(n_kv):
        kh, vh = _stored64(k[:, h]), _stored64(v[:, h])
        s = (q[h * G:(h + 1) * G].double() @ kh.T) / math.sqrt(D)
        out.append(torch.softmax(s, -1) @ vh)
    return torch.cat(out)


def _rope64(x, w, ang_cos, ang_sin, interleaved):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
    half = ang_cos.shape[-1]
    z = torch.complex(ang_cos.double(), ang_sin.double())[:, None]
    y = x.clone()
    i = torch.arange(half, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    r = torch.complex(x[..., first], x[..., second]) * z
    y[..., first], y[..., second] = r.real, r.imag
    return y


def _sample64(x, u, T, k, p, min_p):
    """One row, on the host."""
    best = x.max()
    if T <= 0:
        return int(np.flatnonzero(x == best)[0])
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    w = np.exp((x[order] - best) / T)
    n = len(w)
    if p < 1:
        run = np.cumsum(w)
        n = min(n, int(np.searchsorted(run, p * run[-1])) + 1)
    kept = order[:n][w[:n] >= min_p]
    kept.sort()
    run = np.cumsum(np.exp((x[kept] - best) / T))
    return int(kept[min(int(np.searchsorted(run, u * run[-1], side="right")), len(kept) - 1)])


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "rope":
        cos, sin = s["cos"][s["pos"]], s["sin"][s["pos"]]
        return tuple(_rope64(x, w, cos, sin, case["interleaved"]) for x, w in zip((s["q"], s["k"]), s["w"]))
    if kind == "sample":
        x, u, rows = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy(), {k: v.double().cpu().numpy() for k, v in s["rows"].items()}
        return torch.tensor([_sample64(x[b], u[b], rows["temperature"][b], int(rows["top_k"][b]), rows["top_p"][b], rows["min_p"][b]) for b in range(case["B"])], device="cuda")
    if kind == "prompt":
        return _stored64(s["k"]), _stored64(s["v"])
    if kind == "attend":
        out = [_attend64(s["q"][case["B"] - 1 - i], k, v) for i, k, v in s["contexts"]()]
        return torch.stack(out[::-1])
    ks = [[k] for k, _ in s["prompts"]]
    vs = [[v] for _, v in s["prompts"]]
    out = []
    for q, k, v in s["new"]:
        for b in range(case["B"]):
            ks[b].append(k[b:b + 1])
            vs[b].append(v[b:b + 1])
        out.append(torch.stack([_attend64(q[b], torch.cat(ks[b]), torch.cat(vs[b])) for b in range(case["B"])]))
    return out
