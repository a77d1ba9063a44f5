"""Rotary positions with several axes, with the KV-cache slot write, for packed new tokens.

The reference's RoPE (kernels/rope.py:9-44) and its slot writes share one counter, as
``kv_cache.rope_and_store`` does; here a token's positions (time, height, width of an image or
video, or one position that an eviction has set apart from the slot) are given, and its slot
follows from the cache's lengths.
"""

from __future__ import annotations

from typing import Sequence

import torch

from fast_infer_b200 import _lib
from fast_infer_b200._runtime import device_errors, error_word, stream_of, with_device
from fast_infer_b200.kernels.attention import (_DTYPES, BLOCK_SIZE, CODE_DTYPES, HEAD_DIM,
                                               _batch_args, _check_codes, _check_pages, _check_rows,
                                               _check_scales, _tma_ready)


def rope_axes_store(qkv: torch.Tensor, num_q_heads: int, cos_table: torch.Tensor,
                    sin_table: torch.Tensor, positions: torch.Tensor, sections: Sequence[int],
                    k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    block_size: int, cu_seqlens: torch.Tensor, context_lens: torch.Tensor,
                    q_out: torch.Tensor = None, *, k_scale: torch.Tensor = None,
                    v_scale: torch.Tensor = None) -> torch.Tensor:
    """Rotate q and k of packed new tokens and write k and v to their cache slots, in one launch.

    qkv: [total_tokens, (nq + 2 * nkv) * 128] fp16 or bf16 (q | k | v heads). positions: int32
    [axes, total_tokens] on the device (1 to 4 axes); sections: how many of the 64 frequencies, in
    order, use each axis. cos_table, sin_table: fp32 [rows, 128], indexed by position. k_cache,
    v_cache, block_table, cu_seqlens, context_lens: as in ``paged_chunk_attention``, which takes
    them next; new token i of sequence b is stored at slot ``context_lens[b] - n_b + i``.

    With k_scale and v_scale (fp32 [num_blocks, nkv, 64]) the caches hold 8-bit codes, int8 or
    float8_e4m3fn: every row of 128 of k (rotated, from its fp32 values) and v is written as codes
    Q * x / max|x| (Q = 127 or 448; nearest, ties to even) with the scale max|x| / Q beside it, 0 for a
    row of zeros, NaN for a row that holds NaN or an infinity. ``paged_tree_attention`` and ``read_kv``
    take them.

    The rotation is the rotate-half form in fp32, rounded once. Returns the rotated q
    [total_tokens, nq, 128] (``q_out`` if given; rows outside every sequence are not written). A token
    with a position outside the tables is skipped, and one whose slot has no page is not stored, which
    only device checks (``FAST_INFER_B200_CHECK=1``) report, with a RuntimeError.
    """
    _check_rows("qkv", qkv)
    num_blocks, _, nkv, _ = _check_pages(k_cache, v_cache, k_scale, v_scale, qkv)
    if num_q_heads < 1 or qkv.dim() != 2 or qkv.shape[1] != (num_q_heads + 2 * nkv) * HEAD_DIM:
        raise ValueError("qkv must be [total_tokens, (num_q_heads + 2 * num_kv_heads) * head_dim]")
    total, device = qkv.shape[0], qkv.device
    sections = [int(s) for s in sections]
    if (not isinstance(positions, torch.Tensor) or positions.device != device
            or positions.shape != (len(sections), total)):
        raise ValueError("positions must be an [axes, total_tokens] int32 tensor on qkv's device, "
                         "an axis for each section")
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != HEAD_DIM // 2:
        raise ValueError(f"sections must be 1 to 4 counts that add up to {HEAD_DIM // 2}")
    for name, t in (("cos_table", cos_table), ("sin_table", sin_table)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != device:
            raise ValueError(f"{name} must be a float32 [max_pos, {HEAD_DIM}] table on qkv's device")
    table, steps = cos_table.shape, cos_table.stride()
    if (len(table) != 2 or table[0] == 0 or table[1] != HEAD_DIM or steps[1] != 1
            or sin_table.shape != table or sin_table.stride() != steps):
        raise ValueError(f"cos_table and sin_table must be [max_pos, {HEAD_DIM}] with unit innermost "
                         "stride, laid out alike")
    batch, cu, ctx, bt = _batch_args(device, block_table, block_size, k_cache, cu_seqlens,
                                     context_lens)
    if q_out is None:
        q_out = torch.empty(total, num_q_heads, HEAD_DIM, dtype=qkv.dtype, device=device)
    elif (q_out.shape != (total, num_q_heads, HEAD_DIM) or q_out.dtype != qkv.dtype
          or q_out.device != device or not _tma_ready(q_out)):
        raise ValueError("q_out must be [total_tokens, num_q_heads, head_dim] like qkv, 16-byte "
                         "aligned")
    if batch == 0 or total == 0:
        return q_out
    x = qkv if _tma_ready(qkv) else qkv.clone(memory_format=torch.contiguous_format)
    pos = positions if positions.dtype == torch.int32 else positions.to(torch.int32)
    if pos.stride()[1] != 1:
        pos = pos.contiguous()
    row_stride = steps[0] if table[0] > 1 else HEAD_DIM
    lib = _lib.load()
    with with_device(device):
        err = error_word(device)
        places = (cos_table.data_ptr(), sin_table.data_ptr(), pos.data_ptr(), cu.data_ptr(),
                  ctx.data_ptr(), bt.data_ptr(), total, batch, num_q_heads, nkv, HEAD_DIM,
                  len(sections), _lib.strides(*sections), pos.stride()[0], table[0], row_stride,
                  num_blocks, block_size, bt.shape[1], _lib.strides(*x.stride()),
                  _lib.strides(*q_out.stride()), _lib.strides(*k_cache.stride()),
                  _lib.strides(*v_cache.stride()))
        tail = (err.data_ptr() if err is not None else None, stream_of(device))
        if k_scale is None:
            st = lib.fi_rope_axes_store(
                x.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), *places,
                _lib.strides(*bt.stride()), _DTYPES[qkv.dtype], *tail)
        else:
            st = lib.fi_rope_axes_store8(
                x.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                k_scale.data_ptr(), v_scale.data_ptr(), *places, _lib.strides(*k_scale.stride()),
                _lib.strides(*v_scale.stride()), _lib.strides(*bt.stride()), _DTYPES[qkv.dtype],
                CODE_DTYPES[k_cache.dtype], *tail)
        _lib.check(st, "rope_axes_store")
        device_errors(err, "rope_axes_store")
    return q_out


def read_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
            v_scale: torch.Tensor, block_table: torch.Tensor, block_size: int,
            cu_seqlens: torch.Tensor, context_lens: torch.Tensor, total_tokens: int, *,
            dtype: torch.dtype = torch.float16):
    """Read cached tokens back from pages of 8-bit codes, as 16-bit values.

    k_cache, v_cache: [num_blocks, 64, nkv, 128] int8 or float8_e4m3fn; k_scale, v_scale: fp32
    [num_blocks, nkv, 64]; block_table, cu_seqlens, context_lens: as in ``rope_axes_store``, with
    total_tokens (host int) rows in all: row t of sequence b is its cached token ``context_lens[b] -
    n_b + t`` (with n_b = context_lens[b], the whole sequence). Returns k and v, [total_tokens, nkv,
    128] of ``dtype`` (fp16 or bf16): code * scale in fp32, rounded once. Rows outside every sequence
    are not written, and one whose slot has no page is zero, which only device checks
    (``FAST_INFER_B200_CHECK=1``) report, with a RuntimeError.
    """
    if not isinstance(k_cache, torch.Tensor):
        raise TypeError("k_cache must be a torch.Tensor")
    if not k_cache.is_cuda:
        raise ValueError("k_cache must be a CUDA tensor (fast_infer_b200 has no CPU path)")
    if k_cache.dtype not in CODE_DTYPES:
        raise TypeError(f"k_cache must be int8 or float8_e4m3fn, got {k_cache.dtype}")
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be float16 or bfloat16, got {dtype}")
    shape, device = k_cache.shape, k_cache.device
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _check_codes(name, t, k_cache, shape, k_cache.dtype)
    num_blocks, _, nkv, _ = shape
    _check_scales(k_cache, k_scale, v_scale, (num_blocks, nkv, BLOCK_SIZE))
    batch, cu, ctx, bt = _batch_args(device, block_table, block_size, k_cache, cu_seqlens,
                                     context_lens)
    total = int(total_tokens)
    if total < 0:
        raise ValueError("total_tokens must not be negative")
    k_out = torch.empty(total, nkv, HEAD_DIM, dtype=dtype, device=device)
    v_out = torch.empty_like(k_out)
    if batch == 0 or total == 0:
        return k_out, v_out
    with with_device(device):
        err = error_word(device)
        st = _lib.load().fi_read_kv8(
            k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            k_out.data_ptr(), v_out.data_ptr(), cu.data_ptr(), ctx.data_ptr(), bt.data_ptr(), total,
            batch, nkv, HEAD_DIM, num_blocks, block_size, bt.shape[1],
            _lib.strides(*k_cache.stride()), _lib.strides(*v_cache.stride()),
            _lib.strides(*k_scale.stride()), _lib.strides(*v_scale.stride()),
            _lib.strides(*k_out.stride()), _lib.strides(*v_out.stride()),
            _lib.strides(*bt.stride()), _DTYPES[dtype], CODE_DTYPES[k_cache.dtype],
            err.data_ptr() if err is not None else None, stream_of(device))
        _lib.check(st, "read_kv")
        device_errors(err, "read_kv")
    return k_out, v_out
