"""Norms of queries and keys for each head, and their rotation by position, in one launch."""
from __future__ import annotations
import torch
from . import _lib

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _rows(x: torch.Tensor, n: int) -> torch.Tensor:
    """x [., heads, D] as the kernel reads it: channels next to each other, tokens and heads any multiple of n elements (16 bytes) apart; others are copied."""
    shape, stride = x.shape, x.stride()
    if stride[2] == 1 and (shape[1] == 1 or stride[1] % n == 0) and (shape[0] == 1 or stride[0] % n == 0) and x.data_ptr() % 16 == 0: return x
    return x.clone(memory_format=torch.contiguous_format)


def _aligned(x: torch.Tensor) -> torch.Tensor:
    return x if x.is_contiguous() and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """q [N, n_q, D], k [N, n_kv, D] (bf16, fp16 or fp32; D 64, 128 or 256; any strides of whole 16 bytes between tokens and heads, such as views of a fused
    projection's output) -> new contiguous tensors of their shapes:

      y = x * rsqrt(mean(x^2) + eps) * weight     over the D channels of a head; weights [D] or [heads, D] of q's type, for both or for neither (then y = x)
      of the first R channels the pairs (p, p + R/2), or (2p, 2p + 1) if interleaved, become (y1 cos - y2 sin, y2 cos + y1 sin); the rest stays y

    with row positions[token] (int64 or int32 [N]) of cos, sin (fp32 [max_pos, R/2], R a multiple of 16).  A token whose position the tables do not have becomes NaN.
    In 32 bits, rounded once.  One launch, no wait, no backward pass."""
    out = (_lib._calls or _lib.calls()).norm_rope(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved, _lib.stream)
    if out is not None: return out
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or q.dtype != k.dtype or q.dtype not in TYPES:
        raise RuntimeError(f"qk_norm_rope expects q [N, n_q, D] and k [N, n_kv, D] of one type, bf16, fp16 or fp32, got {q.dtype} {list(q.shape)} and {k.dtype} {list(k.shape)}")
    N, n_q, D = q.shape
    n_k = k.shape[1]
    if D not in (64, 128, 256) or n_q < 1 or n_k < 1: raise RuntimeError(f"qk_norm_rope expects heads of 64, 128 or 256 channels, got {list(q.shape)} and {list(k.shape)}")
    if positions.dtype not in (torch.int64, torch.int32) or tuple(positions.shape) != (N,): raise RuntimeError(f"qk_norm_rope expects positions int64 or int32 [{N}], got {positions.dtype} {list(positions.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] < 1 or not 16 <= 2 * cos.shape[1] <= D or cos.shape[1] % 8:
        raise RuntimeError(f"qk_norm_rope expects cos, sin fp32 [max_pos, R/2], R a multiple of 16 up to {D}, got {cos.dtype} {list(cos.shape)} and {sin.dtype} {list(sin.shape)}")
    if (q_weight is None) != (k_weight is None): raise RuntimeError("qk_norm_rope expects weights for both q and k or for neither")
    if q_weight is not None:
        for w, heads in ((q_weight, n_q), (k_weight, n_k)):
            if w.dtype != q.dtype or tuple(w.shape) not in ((D,), (heads, D)): raise RuntimeError(f"qk_norm_rope expects weights {q.dtype} [{D}] or [{heads}, {D}], got {w.dtype} {list(w.shape)}")
    _lib.no_backward("qk_norm_rope", q, k, cos, sin, q_weight, k_weight)
    with _lib.on_device(q, k, positions, cos, sin, q_weight, k_weight):
        q_out, k_out = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k))
        if N == 0: return q_out, k_out
        per = 16 // q.element_size()
        q, k, positions, cos, sin = _rows(q, per), _rows(k, per), positions.contiguous(), _aligned(cos), _aligned(sin)
        if q_weight is not None: q_weight, k_weight = _aligned(q_weight), _aligned(k_weight)
        at = lambda x, dim: x.stride(dim) if x.shape[dim] > 1 else 0
        _lib.call("gaac_qk_norm_rope", TYPES[q.dtype], q, k, at(q, 0), at(q, 1), at(k, 0), at(k, 1), N, n_q, n_k, D, 2 * cos.shape[1], q_weight, k_weight,
                  D if q_weight is not None and q_weight.dim() == 2 else 0, D if k_weight is not None and k_weight.dim() == 2 else 0, float(eps), positions,
                  int(positions.dtype == torch.int64), cos, sin, cos.shape[0], int(interleaved), q_out, k_out, _lib.stream)
        return q_out, k_out
