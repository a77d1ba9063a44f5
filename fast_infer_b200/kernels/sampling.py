"""Sampling of tokens from logits (the reference takes the greatest logit on the host)."""

from __future__ import annotations

import torch

from fast_infer_b200 import _lib
from fast_infer_b200._runtime import stream_of, with_device

_LOGITS = {torch.float16: _lib.FI_DTYPE_F16, torch.bfloat16: _lib.FI_DTYPE_BF16,
           torch.float32: _lib.FI_DTYPE_F32}
MAX_VOCAB = 262144


def _per_row(name: str, value, dtype: torch.dtype, rows: int, device: torch.device):
    """(tensor or None, scalar) of a setting given for all rows or for each."""
    if not isinstance(value, torch.Tensor):
        return None, value
    if value.shape != (rows,) or value.device != device:
        raise ValueError(f"{name} must be a number or a [rows] tensor on the logits' device")
    if value.dtype != dtype:
        if dtype == torch.int32:
            value = value.to(torch.int64).clamp(0, MAX_VOCAB)  # (no wrap at 2^32; below 0 is all)
        value = value.to(dtype)
    return value.contiguous(), 0


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, *, top_k=0, top_p=1.0,
                  min_p=0.0, out: torch.Tensor = None) -> torch.Tensor:
    """One token per row of logits, from a given uniform number.

    logits: [rows, vocab] fp16, bf16 or fp32 (any row stride; at most 262144 tokens); u: fp32 [rows]
    in [0, 1). temperature, top_k, top_p, min_p: numbers, or tensors of one value per row (fp32,
    top_k int32). With ``w = exp((logit - max) / temperature)`` and tokens in the order of their
    logits, ties by index: top_k keeps the first ``top_k`` (0: all), top_p < 1 those of them before
    which the mass is below ``top_p`` times the mass of them all (the first always stays), min_p those
    with ``w >= min_p`` (min_p in [0, 1]). The token is the first index at which the running sum of
    kept ``w`` is above ``u`` times their whole sum. Weights are rounded to whole units of 2^-45 (of the
    greatest) and added exactly, so shares are off by at most vocab * 2^-46 (3.7e-9 for the largest).
    temperature 0 takes the first of the greatest logits.

    A logit of -inf hides its token. A row that holds NaN or +inf, or nothing above -inf, gives -1.
    Returns int32 [rows] (``out`` if given).
    """
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a torch.Tensor")
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (fast_infer_b200 has no CPU path)")
    if logits.dtype not in _LOGITS:
        raise TypeError(f"logits must be float16, bfloat16 or float32, got {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, vocab]")
    rows, vocab = logits.shape
    device = logits.device
    if vocab > MAX_VOCAB:
        raise ValueError(f"at most {MAX_VOCAB} tokens a row, got {vocab}")
    if (not isinstance(u, torch.Tensor) or u.shape != (rows,) or u.dtype != torch.float32
            or u.device != device):
        raise ValueError("u must be a [rows] float32 tensor on the logits' device")
    t_rows, t = _per_row("temperature", temperature, torch.float32, rows, device)
    k_rows, k = _per_row("top_k", top_k, torch.int32, rows, device)
    p_rows, p = _per_row("top_p", top_p, torch.float32, rows, device)
    m_rows, m = _per_row("min_p", min_p, torch.float32, rows, device)
    if t_rows is None and not 0.0 <= t < float("inf"):
        raise ValueError(f"temperature must be finite and not negative, got {t}")
    if k_rows is None and k < 0:
        raise ValueError(f"top_k must not be negative, got {k}")
    if p_rows is None and not 0.0 <= p <= 1.0 or m_rows is None and not 0.0 <= m <= 1.0:
        raise ValueError(f"top_p and min_p must be in [0, 1], got {p} and {m}")
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=device)
    elif (out.shape != (rows,) or out.dtype != torch.int32 or out.device != device
          or not out.is_contiguous()):
        raise ValueError("out must be a contiguous [rows] int32 tensor on the logits' device")
    if rows == 0:
        return out
    x = logits if logits.stride(1) == 1 or vocab == 1 else logits.contiguous()
    u = u.contiguous()
    with with_device(device):
        st = _lib.load().fi_sample_tokens(
            x.data_ptr(), u.data_ptr(), *(None if r is None else r.data_ptr()
                                          for r in (t_rows, k_rows, p_rows, m_rows)),
            float(t), min(int(k), MAX_VOCAB), float(p), float(m), out.data_ptr(), rows, vocab,
            x.stride(0) if rows > 1 else vocab, _LOGITS[x.dtype], stream_of(device))
        _lib.check(st, "sample_tokens")
    return out
