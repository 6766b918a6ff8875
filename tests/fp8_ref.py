"""Definitions of rows in 8 bits, norm, products and log probabilities in 64 bits, with the largest errors that the kernels' roundings may make."""
import torch

BLOCK = 128


def exponents(x):
    """E of every block of x [M, K] (fp64): the smallest with max |x| <= 448 * 2^E, from -117 to 119."""
    M, K = x.shape
    b = torch.cat([x, x.new_zeros(M, -K % BLOCK)], 1).view(M, -1, BLOCK)
    top = b.abs().amax(-1)
    E = torch.full_like(top, 119.0)
    for e in range(118, -118, -1): E = torch.where(top <= 448 * 2.0 ** e, float(e), E)
    return b, E, torch.isfinite(top)


GRID = torch.tensor([(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127], dtype=torch.float64)      # e4m3's values from 0 to 448, by code


def stored(x):
    """fp64 values that 8 bits hold of x [M, K] (on the CPU), found by distance: the nearest, of two the one with the even code."""
    x = x.detach().double().cpu()
    b, E, fine = exponents(x)
    s = torch.exp2(E).unsqueeze(-1)
    y = (b.abs() / s).nan_to_num(0.0, 0.0, 0.0)
    hi = torch.bucketize(y, GRID).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    d_lo, d_hi = y - GRID[lo], GRID[hi] - y
    code = torch.where(d_lo < d_hi, lo, torch.where(d_hi < d_lo, hi, torch.where(lo % 2 == 0, lo, hi)))
    v = GRID[code] * s * torch.where(torch.signbit(b), -1.0, 1.0)
    return torch.where(fine.unsqueeze(-1), v, torch.nan).flatten(1)[:, :x.shape[1]]


def half_step(y):
    """Half the distance of the grid's values around each element of y [M, K]: what a nearest value may be off by."""
    b, E, _ = exponents(y)
    s = torch.exp2(E).unsqueeze(-1)
    e = torch.floor(torch.log2((b.abs() / s).clamp(min=2.0 ** -6)))
    return (torch.exp2(e - 4) * s).flatten(1)[:, :y.shape[1]]


def norm(x, weight, eps, residual=None):
    """(y, h) in 64 bits."""
    h = x.detach().double().cpu()
    if residual is not None: h = h + residual.detach().double().cpu()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.detach().double().cpu(), h


def cut(x, w):
    """What the 8-bit product may lose of x w^T (values [M, K], [N, K]): it adds the products of eight consecutive elements as whole multiples of 2^-13 of 2^e, e the largest sum of the exponents of two factors
    among the eight, cutting what is below; the largest product itself (8 bits) loses nothing, the other seven less than one such multiple each."""
    def power(v):      # of the largest factor of each eight: 2^exponent.  (An element whose code is below the grid's normal numbers has the power of the smallest of them, 2^-6 of the block's.)
        v = torch.cat([v, v.new_zeros(v.shape[0], -v.shape[1] % BLOCK)], 1)
        _, E, _ = exponents(v)
        top = v.view(v.shape[0], -1, BLOCK // 8, 8).abs().amax(-1)
        floor = torch.exp2(E - 6).unsqueeze(-1)
        return torch.where(top > 0, torch.exp2(torch.floor(torch.log2(torch.maximum(top, floor)))), 0.0).flatten(1)
    return 7 * 2.0 ** -13 * (power(x) @ power(w).T)


def product(x, w, dtype, exact=None):
    """x [M, K], w [N, K] (values) -> (x w^T, largest error).  A sum of K products in 32 bits: each addition off by at most 2^-23 of the sum of magnitudes (as if the matrix unit cut instead of rounding);
    for outputs of 16 bits what the 8-bit product cuts; then one rounding of the type."""
    x, w = x.double().cpu(), w.double().cpu()
    y, mag = x @ w.T, x.abs() @ w.abs().T
    f = torch.finfo(dtype)
    loss = 0.0 if (dtype == torch.float32 if exact is None else exact) else cut(x, w)
    return y, loss * 1.01 + x.shape[1] * 2.0 ** -23 * mag + f.eps / 2 * y.abs() * 1.01 + f.smallest_normal * f.eps


def gated(x, gate, up, dtype):
    """silu(x gate^T) * (x up^T) -> (y, largest error): those of both sums (silu's slope is at most 1.1), silu itself a few roundings of 2^-22, its exponential's argument |g| * 2^-23."""
    (g, dg), (u, du) = (product(x, w, torch.float32, exact=dtype == torch.float32) for w in (gate, up))
    a = g * torch.sigmoid(g)
    y = a * u
    f = torch.finfo(dtype)
    return y, 1.1 * dg * (u.abs() + du) + a.abs() * du + (2.0 ** -20 + g.abs() * 2.0 ** -22) * y.abs() + f.eps / 2 * y.abs() * 1.01 + f.smallest_normal * f.eps


def logprobs(logits, tokens, top):
    """(logprob, rank, entropy, top_logprobs, top_tokens, tolerance of a log probability of size p, of the entropy), fp64 / int64 on the CPU.

    e^d is off by 1.2 |d| 2^-24 of itself, 2^-19 for |d| up to 26 (what lies farther below adds less than 2^-19 of the sum, even 2^18 times); a sum passes 16 + 6 + 8 additions and one for each segment, 2^-24 each, at most 2^-18 for the segments of the tests; so the sum's logarithm is off by 2^-17; differences and
    the result are rounded to 24 bits.  The entropy's second term is such a sum of e^d d, over the first."""
    x = logits.detach().double().cpu()
    x = torch.where(x.isnan(), -torch.inf, x)
    B, V = x.shape
    best = x.amax(-1, keepdim=True)
    d = torch.where(x == best, 0.0, x - best)
    d = torch.where(best == -torch.inf, torch.nan, d)
    S = torch.exp(d).sum(-1, keepdim=True)
    lp = d - torch.log(S)
    p = lp.exp()
    far = torch.where(p > 0, p * d.abs(), 0.0).sum(-1)
    entropy = torch.log(S)[:, 0] + far
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    place = torch.empty_like(order).scatter_(1, order, torch.arange(V).expand(B, V))
    t = tokens.cpu()
    inside = (t >= 0) & (t < V)
    at = t.clamp(0, V - 1)[:, None]
    value = torch.where(inside, lp.gather(1, at)[:, 0], torch.nan)
    entropy = torch.where(best[:, 0] == -torch.inf, torch.nan, entropy)
    tol = lambda v: 2.0 ** -17 + 2.0 ** -21 * v.abs().nan_to_num(0, 0, 0)
    return value, torch.where(inside, place.gather(1, at)[:, 0], -1), entropy, lp.gather(1, order[:, :top]), order[:, :top], tol, 2.0 ** -17 * (2 + 2 * far) + 2.0 ** -21 * torch.log(S)[:, 0]
