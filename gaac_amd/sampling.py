"""Sampling of one token per row from logits, with given random numbers."""
from __future__ import annotations
import torch
from . import _lib
from .rope import TYPES

MAX_VOCAB = (1 << 20) - 16


def work_bytes(B: int, V: int) -> int:
    """Scratch of a call: none for rows of one segment of 4096 logits, otherwise for each of up to 1024 rows at a time two words for each segment, 2048 bins of 12 bytes, 8192
    candidates, two counters."""
    segments = -(-(V + 7) // 4096)
    return 0 if segments == 1 else min(B, 1024) * (16 * segments + 12 * 2048 + 8 * 8192 + 16)


def _setting(name: str, x, B: int, dtype, like: torch.Tensor):
    """(tensor or None, number) of a setting that is a number or one per row."""
    if not isinstance(x, torch.Tensor): return None, x
    if tuple(x.shape) != (B,) or x.dtype != dtype: raise RuntimeError(f"sample expects {name} as a number or {dtype} [{B}], got {x.dtype} {list(x.shape)}")
    return x.contiguous(), 0


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """logits [B, V] (bf16, fp16 or fp32, rows any stride apart), u fp32 [B] in [0, 1) -> token int64 [B].  Each setting is a number or a tensor [B] (fp32; top_k int32).

      w_i = exp((x_i - max) / temperature); the order of tokens is x descending, then index ascending
      kept: the first top_k of the order (0 or less: all); of these the shortest prefix whose sum of w is at least top_p times theirs, and at least one token
            (1 or more: all); of these the ones with w >= min_p, the maximum having 1 (0 or less: all)
      token: the first i, in the order of the vocabulary, at which the running sum of the kept w exceeds u times their total

    A temperature that is not positive: the first maximum.  A token whose logit is -inf or NaN never comes; -1 for a row that has nothing else.  An infinite
    maximum: evenly among the tokens that have it.  u outside [0, 1) counts as the nearest number inside, NaN as 0.  Weights are rounded to multiples of 2^-43
    of the largest one, and what is rounded is added exactly: a sum over n tokens is off by at most n * 2^-44 of the largest weight (2^-24 for a vocabulary of 2^20), the same in
    any order, and a token whose weight is below 2^-44 never comes.  One launch for vocabularies up to 4089, otherwise at most three for every 1024 rows; no wait."""
    out = (_lib._calls or _lib.calls()).draw(logits, u, temperature, top_k, top_p, min_p, _lib.stream)
    if out is not None: return out
    if logits.dim() != 2 or logits.dtype not in TYPES or not 1 <= logits.shape[1] <= MAX_VOCAB:
        raise RuntimeError(f"sample expects logits bf16, fp16 or fp32 [B, V], V up to {MAX_VOCAB}, got {logits.dtype} {list(logits.shape)}")
    B, V = logits.shape
    if u.dtype != torch.float32 or tuple(u.shape) != (B,): raise RuntimeError(f"sample expects u fp32 [{B}], got {u.dtype} {list(u.shape)}")
    (t_rows, t), (k_rows, k), (p_rows, p), (m_rows, m) = (_setting(name, x, B, dtype, logits) for name, x, dtype in (
        ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)))
    with _lib.on_device(logits, u, t_rows, k_rows, p_rows, m_rows):
        out = torch.empty(B, dtype=torch.int64, device=logits.device)
        if B == 0: return out
        work = torch.empty(work_bytes(B, V), dtype=torch.uint8, device=logits.device)
        if V > 1 and logits.stride(1) != 1 or B > 1 and logits.stride(0) < 0: logits = logits.contiguous()
        _lib.call("gaac_sample", TYPES[logits.dtype], logits, logits.stride(0) if B > 1 else 0, B, V, u.contiguous(), t_rows, float(t), k_rows, max(0, min(int(k), V)), p_rows, float(p), m_rows, float(m), work, work.numel(), out, _lib.stream)
        return out
