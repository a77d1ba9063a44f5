"""Eviction from the paged KV cache by accumulated attention weight (no counterpart in the
reference). ``kernels.attention.attention_mass`` gives the weights; ``KVCache.evict`` does the same
as ``evict_tokens`` in place, with the cache's own bookkeeping.
"""

from __future__ import annotations

import torch

from fast_infer_b200 import _lib
from fast_infer_b200._runtime import device_errors, error_word, stream_of, with_device

HEAD_DIM = 128
BLOCK_SIZE = 64


def _check_pools(what: str, k: torch.Tensor, v: torch.Tensor) -> None:
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{what}{name} must be a CUDA tensor (fast_infer_b200 has no CPU path)")
        if t.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"{what}{name} must be float16 or bfloat16, got {t.dtype}")
        shape = t.shape
        if len(shape) != 5 or shape[2] != BLOCK_SIZE or shape[4] != HEAD_DIM:
            raise ValueError(f"{what}{name} must be [layers, num_blocks, {BLOCK_SIZE}, num_heads, "
                             f"{HEAD_DIM}]")
    if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
        raise ValueError(f"{what}k and {what}v must have the same shape, type and device")


def _check_table(name: str, t: torch.Tensor, batch: int, device: torch.device) -> None:
    shape = t.shape if isinstance(t, torch.Tensor) else ()
    if (len(shape) != 2 or shape[0] < batch or shape[1] == 0 or t.dtype != torch.int32
            or t.device != device):
        raise ValueError(f"{name} must be a [>= batch, max_blocks] int32 tensor on the cache's device")


def evict_tokens(k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, mass: torch.Tensor, budget: int, *, recent: int = 0,
                 sinks: int = 0, out=None):
    """Keep at most ``budget`` cached tokens per (layer, sequence, KV head): the first ``sinks``,
    the last ``recent`` and, of those between, the ones with the greatest ``mass`` (ties: lowest
    index; negative and NaN count as 0). They keep their order and move to slots 0, 1, ...

    k, v: [layers, num_blocks, 64, num_heads, 128] fp16 or bf16 pools (``KVCache.k`` / ``.v``);
    block_table: [>= batch, max_blocks] int32; seq_lens: [batch] int32 on the device; mass: fp32
    [layers, batch, num_heads, capacity]. By default in place: afterwards sequence b holds
    min(seq_lens[b], budget) tokens in its first pages; pages must not be shared between
    sequences. ``out`` = (k_out, v_out, block_table_out) writes them to those pools' pages instead
    and leaves the source as it was (the pages read and written must not overlap).

    ``capacity`` and the block table have to reach as far as every sequence: a longer one counts as if
    it ended there (``recent`` with it), and its newest tokens are lost. Lengths are on the device, so
    only device checks (``FAST_INFER_B200_CHECK=1``) report that, with a RuntimeError.

    Returns (kept, mass_out), both [layers, batch, num_heads, budget]: the old slots that stay,
    ascending (int32, -1 past the last), and their mass (0 past the last).
    """
    _check_pools("", k, v)
    layers, num_blocks, _, heads, _ = k.shape
    device = k.device
    if not isinstance(seq_lens, torch.Tensor) or seq_lens.dim() != 1 or seq_lens.device != device:
        raise ValueError("seq_lens must be a [batch] int32 tensor on the cache's device")
    batch = seq_lens.numel()
    _check_table("block_table", block_table, batch, device)
    if (not isinstance(mass, torch.Tensor) or mass.dim() != 4
            or mass.shape[:3] != (layers, batch, heads) or mass.dtype != torch.float32
            or mass.device != device):
        raise ValueError("mass must be a [layers, batch, num_heads, capacity] float32 tensor on the "
                         "cache's device")
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError(f"needs budget >= 1 and recent + sinks <= budget, got {budget}, {recent}, "
                         f"{sinks}")
    if out is None:
        k_out, v_out, table_out = k, v, block_table
    else:
        k_out, v_out, table_out = out
        _check_pools("out ", k_out, v_out)
        out_shape = k_out.shape
        if (out_shape[0] != layers or out_shape[3] != heads or k_out.dtype != k.dtype
                or k_out.device != device):
            raise ValueError("out pools need the same layers, heads, type and device as k and v")
        _check_table("out block_table", table_out, batch, device)
    if budget > table_out.shape[1] * BLOCK_SIZE:
        raise ValueError(f"budget {budget} does not fit the block table")
    shape = (layers, batch, heads, budget)
    kept = torch.empty(shape, dtype=torch.int32, device=device)
    mass_out = torch.empty(shape, dtype=torch.float32, device=device)
    if kept.numel() == 0:
        return kept, mass_out
    lens = seq_lens if seq_lens.dtype == torch.int32 else seq_lens.to(torch.int32)
    lens, mass = lens.contiguous(), mass.contiguous()
    lib = _lib.load()
    with with_device(device):
        err = error_word(device)
        st = lib.fi_kv_evict(
            k.data_ptr(), v.data_ptr(), block_table.data_ptr(), lens.data_ptr(), mass.data_ptr(),
            k_out.data_ptr(), v_out.data_ptr(), table_out.data_ptr(), kept.data_ptr(),
            mass_out.data_ptr(), layers, batch, heads, HEAD_DIM, num_blocks, k_out.shape[1],
            BLOCK_SIZE, block_table.shape[1], table_out.shape[1], mass.shape[3], budget, recent,
            sinks, _lib.strides(*k.stride()), _lib.strides(*v.stride()),
            _lib.strides(*k_out.stride()), _lib.strides(*v_out.stride()),
            _lib.strides(*block_table.stride()), _lib.strides(*table_out.stride()),
            err.data_ptr() if err is not None else None, stream_of(device))
        _lib.check(st, "evict_tokens")
        device_errors(err, "evict_tokens")
    return kept, mass_out
