"""Definitions of the 4-bit cache, norm + rotation, and sampling in 64 bits, for the tests."""
import math

import numpy as np
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def stored(x):
    """fp64 values that the 4-bit cache holds of x [..., 128] (on the CPU)."""
    x = x.detach().cpu()
    b = x.double().unflatten(-1, (x.shape[-1] // 32, 32))
    top = b.abs().amax(-1, keepdim=True)
    E = torch.full_like(top, -125.0)
    fine = torch.isfinite(top)
    for e in range(-125, 126):      # the smallest E with top < 7 * 2^E, from -125 to 125
        E = torch.where(top >= 7 * 2.0 ** (e - 1), float(e), E) if e > -125 else E
    s = torch.exp2(E)
    y = b.abs() / s
    d = (y.unsqueeze(-1) - GRID).abs()
    near = d.amin(-1, keepdim=True)
    tie = d == near
    even = torch.arange(8) % 2 == 0
    code = torch.where(tie.sum(-1) > 1, (tie & even).float().argmax(-1), tie.float().argmax(-1))
    v = GRID[code] * s * torch.where(torch.signbit(b), -1.0, 1.0)
    return torch.where(fine, v, math.nan).reshape(x.shape)


def attention(q, k, v, scale):
    """q [n_q, 128], k, v [L, n_kv, 128] (values of the cache) -> (output, largest error that the kernel's roundings may make), both fp64 [n_q, 128].

    Roundings: a score is a sum of 128 products in 32 bits (128 * 2^-24 of the sum of their magnitudes) times scale, its exponent two more operations of 2^-24 of
    the largest |score| and exp2 of 2^-22; a weight goes to bf16 (2^-8 of itself); the sums over tokens in 32 bits (2^-24 a token); the output to bf16."""
    q, k, v = q.detach().double().cpu(), k.double().cpu(), v.double().cpu()
    n_q, (L, n_kv, D) = q.shape[0], k.shape
    G = n_q // n_kv
    out, tol = torch.zeros(n_q, D, dtype=torch.float64), torch.zeros(n_q, D, dtype=torch.float64)
    if L == 0: return out, tol
    for h in range(n_kv):
        qh = q[h * G:(h + 1) * G]
        s = qh @ k[:, h].T * scale
        size = (qh.abs() @ k[:, h].abs().T * abs(scale)).amax(-1, keepdim=True)
        p = torch.softmax(s, -1)
        o, mag = p @ v[:, h], p @ v[:, h].abs()
        rel = 2 * (128 + 8) * 2.0 ** -24 * size + 2.0 ** -20 + L * 2.0 ** -24 + 2.0 ** -8
        out[h * G:(h + 1) * G] = o
        tol[h * G:(h + 1) * G] = rel * mag * 1.01 + 2.0 ** -8 * o.abs() + 1e-37
    return out, tol


def norm_rope(x, w, cos, sin, interleaved, eps):
    """x [N, heads, D], cos, sin [N, R/2] -> (y, largest error), fp64.

    Roundings: the sum of squares D * 2^-24, square root, quotient and two products a few 2^-24 of y; the rotation two products and a sum; then one of the type."""
    dtype = x.dtype
    x = x.detach().double().cpu()
    if w is not None: x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.detach().double().cpu()
    half, D = cos.shape[-1], x.shape[-1]
    c, s = cos.double().cpu()[:, None], sin.double().cpu()[:, None]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, mag = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    mag[..., a], mag[..., b] = (x[..., a] * c).abs() + (x[..., b] * s).abs(), (x[..., b] * c).abs() + (x[..., a] * s).abs()
    f = torch.finfo(dtype)
    return y, f.eps / 2 * y.abs() * 1.01 + ((D + 16) * 2.0 ** -24 if w is not None else 4 * 2.0 ** -24) * mag + f.smallest_normal * f.eps


def sample(x, u, T, k, p, min_p):
    """One row, numpy float64 x; u, T, p, min_p floats."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf: return -1
    if not T > 0: return int(np.flatnonzero(x == top)[0])
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - top) / T)))
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0: order = order[:k]
    if p < 1:
        run = np.cumsum(w[order])
        before = np.concatenate([[0.0], run[:-1]])
        keep = before < p * run[-1]
        keep[0] = True
        order = order[keep]
    order = order[w[order] >= min(min_p, 1.0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    u = 0.0 if not u > 0 else u
    at = int(np.searchsorted(run, u * run[-1], side="right"))
    if at >= len(run): at = int(np.flatnonzero(w[kept] > 0)[-1])
    return int(kept[at])
