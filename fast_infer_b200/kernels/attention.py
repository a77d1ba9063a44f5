"""FlashAttention (prefill) and paged attention (decode) on B200 — drop-in module.

Same functions, argument meaning and return conventions as the reference
``kernels/attention.py`` (``flash_attention`` at :80-113, ``paged_attention`` at
:191-233), so ``model.py`` calls this module unchanged. The work runs in the
sm_100a CUDA library (``libfast_infer_b200.so``) reached through its C ABI; there
is no Triton and no CPU path — CPU tensors are rejected.

Backward-compatible extensions:
* ``flash_attention`` also accepts un-expanded GQA K/V (``k.shape[1]`` dividing
  ``q.shape[1]``), so callers can drop the ``repeat_interleave`` of model.py:110-111.
* ``paged_attention`` takes optional per-sequence ``context_lens`` (ragged
  batches) and ``pages_per_split`` (split-KV tuning).

Functions without a reference counterpart, for serving long contexts in chunks (fp16 and
bf16): ``paged_chunk_attention`` (new tokens over the paged cache, with capped scores, a
distance bias, a window or a prefix), ``attention_mass`` (the weight each cached token received) and
``paged_tree_attention`` (trees of drafted tokens, and caches of 8-bit codes).
"""

from __future__ import annotations

import functools

import torch

from fast_infer_b200 import _lib
from fast_infer_b200._runtime import (device_errors, error_word, stream_of, with_device)

HEAD_DIM = 128
BLOCK_SIZE = 64


def _check_cuda_f16(name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (fast_infer_b200 has no CPU path)")
    if t.dtype != torch.float16:
        raise TypeError(f"{name} must be float16, got {t.dtype}")


@functools.lru_cache(maxsize=4096)
def _tma_strides(shape, strides) -> bool:
    if strides[-1] != 1:
        return False
    for i in range(len(strides) - 1):
        if strides[i] % 8 != 0 and shape[i] != 1:
            return False
    return True


def _tma_ready(t: torch.Tensor) -> bool:
    """True if the tensor can be addressed by a TMA map as is: 16-byte aligned base,
    unit innermost stride, every other stride a multiple of 8 elements."""
    return t.data_ptr() % 16 == 0 and _tma_strides(t.shape, t.stride())


def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    sm_scale: float = None) -> torch.Tensor:
    """Causal FlashAttention for the prefill phase.

    q: [batch, num_heads, seq_len, head_dim] fp16 (any strides, e.g. the BHSD view of
    BSHD memory that model.py passes); k, v: [batch, num_kv_heads, seq_len, head_dim]
    with num_kv_heads == num_heads (expanded, as the reference caller passes them) or
    dividing num_heads (GQA, no expansion needed).
    Returns a tensor shaped and strided like ``torch.empty_like(q)``
    (reference attention.py:99).
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_cuda_f16(name, t)
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D [batch, heads, seq_len, head_dim]")
    batch, num_heads, seq_len, head_dim = q.shape
    if head_dim != HEAD_DIM:
        raise ValueError(f"head_dim must be {HEAD_DIM}, got {head_dim}")
    if k.shape != v.shape or k.shape[0] != batch or k.shape[2] != seq_len or k.shape[3] != head_dim:
        raise ValueError(f"k/v shape {tuple(k.shape)}/{tuple(v.shape)} incompatible with q {tuple(q.shape)}")
    num_kv_heads = k.shape[1]
    if num_kv_heads == 0 or num_heads % num_kv_heads != 0:
        raise ValueError(f"num_heads {num_heads} not a multiple of k/v heads {num_kv_heads}")
    if not (q.device == k.device == v.device):
        raise ValueError("q, k, v must be on the same device")
    if sm_scale is None:
        sm_scale = head_dim ** -0.5
    o = torch.empty_like(q)
    if q.numel() == 0:
        return o
    qx = q if _tma_ready(q) else q.contiguous()
    kx = k if _tma_ready(k) else k.contiguous()
    vx = v if _tma_ready(v) else v.contiguous()
    ox = o if _tma_ready(o) else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lib = _lib.load()
    with with_device(q.device):
        err = error_word(q.device)
        st = lib.fi_prefill_fwd(
            qx.data_ptr(), kx.data_ptr(), vx.data_ptr(), ox.data_ptr(),
            batch, num_heads, num_kv_heads, seq_len, head_dim,
            _lib.strides(*qx.stride()), _lib.strides(*kx.stride()),
            _lib.strides(*vx.stride()), _lib.strides(*ox.stride()),
            float(sm_scale), err.data_ptr() if err is not None else None, stream_of(q.device))
        _lib.check(st, "flash_attention")
        device_errors(err, "flash_attention")
    if ox is not o:
        o.copy_(ox)
    return o


def flash_attention_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           cu_seqlens: torch.Tensor, max_seqlen: int,
                           sm_scale: float = None) -> torch.Tensor:
    """Causal prefill over a ragged batch packed along the token axis (extension; the
    reference's ``flash_attention`` takes one shared sequence length).

    q: [total_tokens, num_heads, 128] fp16; k, v: [total_tokens, num_kv_heads, 128];
    sequence b owns tokens [cu_seqlens[b], cu_seqlens[b+1]) (int32 on the device);
    max_seqlen (host int) bounds the lengths. Returns o shaped like q.
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_cuda_f16(name, t)
        if t.dim() != 3 or t.shape[-1] != HEAD_DIM:
            raise ValueError(f"{name} must be [total_tokens, heads, {HEAD_DIM}]")
    total, num_heads, head_dim = q.shape
    if k.shape != v.shape or k.shape[0] != total:
        raise ValueError("k/v must be [total_tokens, num_kv_heads, head_dim] like q")
    num_kv_heads = k.shape[1]
    if num_heads % num_kv_heads != 0:
        raise ValueError(f"num_heads {num_heads} not a multiple of k/v heads {num_kv_heads}")
    if cu_seqlens.dim() != 1 or cu_seqlens.device != q.device:
        raise ValueError("cu_seqlens must be a 1-D int32 tensor on q's device")
    cu = cu_seqlens.to(torch.int32).contiguous()
    batch = cu.numel() - 1
    if sm_scale is None:
        sm_scale = head_dim ** -0.5
    o = torch.empty_like(q)
    if batch <= 0 or total == 0:
        return o
    qx = q if _tma_ready(q) else q.contiguous()
    kx = k if _tma_ready(k) else k.contiguous()
    vx = v if _tma_ready(v) else v.contiguous()
    ox = o if _tma_ready(o) else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lib = _lib.load()
    with with_device(q.device):
        err = error_word(q.device)
        st = lib.fi_prefill_fwd_varlen(
            qx.data_ptr(), kx.data_ptr(), vx.data_ptr(), ox.data_ptr(), cu.data_ptr(), batch,
            num_heads, num_kv_heads, int(max_seqlen), total, head_dim,
            _lib.strides(*qx.stride()), _lib.strides(*kx.stride()),
            _lib.strides(*vx.stride()), _lib.strides(*ox.stride()), float(sm_scale),
            err.data_ptr() if err is not None else None, stream_of(q.device))
        _lib.check(st, "flash_attention_varlen")
        device_errors(err, "flash_attention_varlen")
    if ox is not o:
        o.copy_(ox)
    return o


def paged_attention_workspace_bytes(batch: int, num_q_heads: int, num_kv_heads: int,
                                    max_context_len: int, pages_per_split: int = 0) -> int:
    """Split-KV workspace bytes ``paged_attention`` needs for these sizes."""
    return int(_lib.load().fi_paged_decode_workspace_size(
        batch, num_q_heads, num_kv_heads, HEAD_DIM, max_context_len, BLOCK_SIZE, pages_per_split))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, block_size: int,
                    num_tokens: int,
                    sm_scale: float = None, *,
                    context_lens: torch.Tensor = None,
                    max_context_len: int = None,
                    pages_per_split: int = 0,
                    workspace: torch.Tensor = None) -> torch.Tensor:
    """PagedAttention for the decode phase (one query token per sequence).

    q: [batch, num_q_heads, head_dim] fp16; k_cache, v_cache: [num_blocks, block_size,
    num_kv_heads, head_dim] fp16 (one layer of ``KVCache.k`` / ``.v``); block_table:
    [>= batch, max_blocks_per_seq] int32 with -1 for unused slots; num_tokens: valid
    tokens of every sequence (reference semantics; 0 returns zeros). Pass
    ``context_lens`` ([batch] int32 on the device) for per-sequence lengths instead;
    ``max_context_len`` (host int) then bounds them (default: the block table's span,
    which needs no device sync). ``workspace`` optionally supplies the split-KV
    scratch (uint8, at least ``paged_attention_workspace_bytes`` bytes).
    Returns [batch, num_q_heads, head_dim] fp16 like ``torch.empty_like(q)``.
    """
    if context_lens is None and num_tokens == 0:
        return torch.zeros_like(q)
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)):
        _check_cuda_f16(name, t)
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("expected q [B, Hq, D] and k_cache/v_cache [NB, block_size, Hkv, D]")
    batch, num_q_heads, head_dim = q.shape
    num_blocks, bs, num_kv_heads, d2 = k_cache.shape
    if head_dim != HEAD_DIM or d2 != HEAD_DIM:
        raise ValueError(f"head_dim must be {HEAD_DIM}")
    if block_size != bs or bs != BLOCK_SIZE:
        raise ValueError(f"block_size must be {BLOCK_SIZE} and match k_cache.shape[1]")
    if block_table.dim() != 2 or block_table.shape[0] < batch:
        raise ValueError("block_table must be [>= batch, max_blocks_per_seq]")
    if block_table.device != q.device or k_cache.device != q.device:
        raise ValueError("all tensors must be on the same device")
    if block_table.dtype != torch.int32:
        block_table = block_table.to(torch.int32)
    max_blocks = block_table.shape[1]
    if context_lens is not None:
        if context_lens.dtype != torch.int32:
            context_lens = context_lens.to(torch.int32)
        if context_lens.device != q.device or context_lens.numel() < batch:
            raise ValueError("context_lens must be a [batch] int32 tensor on q's device")
        context_lens = context_lens.contiguous()
        if max_context_len is None:
            max_context_len = max_blocks * block_size
        ntok = 0
    else:
        if num_tokens < 0 or (num_tokens + block_size - 1) // block_size > max_blocks:
            raise ValueError(f"num_tokens {num_tokens} does not fit the block table")
        ntok = int(num_tokens)
        max_context_len = ntok
    if sm_scale is None:
        sm_scale = head_dim ** -0.5
    o = torch.empty_like(q)
    if batch == 0:
        return o
    lib = _lib.load()
    need = int(lib.fi_paged_decode_workspace_size(batch, num_q_heads, num_kv_heads, head_dim,
                                                  max_context_len, block_size, pages_per_split))
    if need > 0:
        if workspace is None or workspace.numel() * workspace.element_size() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    with with_device(q.device):
        err = error_word(q.device)
        st = lib.fi_paged_decode(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(),
            block_table.data_ptr(),
            context_lens.data_ptr() if context_lens is not None else None,
            ntok, int(max_context_len), batch, num_q_heads, num_kv_heads, head_dim,
            num_blocks, block_size, max_blocks,
            _lib.strides(*q.stride()), _lib.strides(*k_cache.stride()),
            _lib.strides(*v_cache.stride()), _lib.strides(*o.stride()),
            _lib.strides(*block_table.stride()), float(sm_scale), int(pages_per_split),
            workspace.data_ptr() if need > 0 else None, need,
            err.data_ptr() if err is not None else None, stream_of(q.device))
        _lib.check(st, "paged_attention")
        device_errors(err, "paged_attention")
    return o


_DTYPES = {torch.float16: _lib.FI_DTYPE_F16, torch.bfloat16: _lib.FI_DTYPE_BF16}
# Codes of an 8-bit cache, and every type of a page pool.
CODE_DTYPES = {torch.int8: _lib.FI_DTYPE_I8, torch.float8_e4m3fn: _lib.FI_DTYPE_E4M3}
POOL_DTYPES = {**_DTYPES, **CODE_DTYPES}


def _int32_on(name: str, t: torch.Tensor, device: torch.device, count: int) -> torch.Tensor:
    if (not isinstance(t, torch.Tensor) or t.device != device or t.dim() != 1
            or t.numel() != count):
        raise ValueError(f"{name} must be a 1-D int32 tensor of {count} values on {device}")
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


@functools.lru_cache(maxsize=4096)
def _cache_shape(shape) -> bool:
    return len(shape) == 4 and shape[3] == HEAD_DIM and 0 not in shape


def _check_cache(name: str, t: torch.Tensor, like: torch.Tensor, shape) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (fast_infer_b200 has no CPU path)")
    if t.dtype != like.dtype:
        raise TypeError(f"{name} must be float16 or bfloat16 like the new tokens, got {t.dtype}")
    if t.device != like.device:
        raise ValueError("all tensors must be on the same device")
    if t.shape != shape or not _cache_shape(shape):
        raise ValueError(f"{name} must be [num_blocks, {BLOCK_SIZE}, num_kv_heads, {HEAD_DIM}]")
    if not _tma_ready(t):
        raise ValueError(f"{name} needs a 16-byte aligned base, unit innermost stride and "
                         "other strides that are multiples of 8")


@functools.lru_cache(maxsize=4096)
def _code_strides(shape, strides) -> bool:
    return strides[-1] == 1 and all(st % 16 == 0 or n == 1 for n, st in zip(shape[:-1], strides))


def _check_codes(name: str, t: torch.Tensor, like: torch.Tensor, shape, dtype) -> None:
    """Like ``_check_cache`` for a pool of 8-bit codes."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"k_cache and v_cache must have the same type, got {dtype} and {t.dtype}")
    if t.device != like.device:
        raise ValueError("all tensors must be on the same device")
    if t.shape != shape or not _cache_shape(shape):
        raise ValueError(f"{name} must be [num_blocks, {BLOCK_SIZE}, num_kv_heads, {HEAD_DIM}]")
    if t.data_ptr() % 16 != 0 or not _code_strides(t.shape, t.stride()):
        raise ValueError(f"{name} needs a 16-byte aligned base, unit innermost stride and "
                         "other strides that are multiples of 16")


def _check_scales(pool: torch.Tensor, k_scale, v_scale, shape) -> None:
    """The scales that go with a pool: fp32 of this shape for codes, none for 16-bit values."""
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if pool.dtype not in CODE_DTYPES:
            if t is not None:
                raise ValueError(f"{name} goes with an int8 or float8_e4m3fn cache only")
        elif (not isinstance(t, torch.Tensor) or t.dtype != torch.float32
              or t.device != pool.device or t.shape != shape):
            raise ValueError(f"{name} must be a float32 tensor {list(shape)} on the cache's device "
                             "([..., num_blocks, num_kv_heads, 64])")


def _check_pages(k_cache, v_cache, k_scale, v_scale, like) -> tuple:
    """Checks of one layer's pages, 16-bit like the rows `like` or codes with scales; their shape."""
    shape = k_cache.shape if isinstance(k_cache, torch.Tensor) else None
    if isinstance(k_cache, torch.Tensor) and k_cache.dtype in CODE_DTYPES:
        for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
            _check_codes(name, t, like, shape, k_cache.dtype)
    else:
        _check_cache("k_cache", k_cache, like, shape)
        _check_cache("v_cache", v_cache, like, shape)
    if k_scale is not None or v_scale is not None or k_cache.dtype in CODE_DTYPES:
        _check_scales(k_cache, k_scale, v_scale, (shape[0], shape[2], BLOCK_SIZE))
    return shape


def _check_rows(name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (fast_infer_b200 has no CPU path)")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float16 or bfloat16, got {t.dtype}")


def _batch_args(device, block_table, block_size, k_cache, cu_seqlens, context_lens):
    """Checks of the packed batch and its block table; (batch, cu, ctx, table) as the library
    takes them."""
    if block_size != BLOCK_SIZE or k_cache.shape[1] != BLOCK_SIZE:
        raise ValueError(f"block_size must be {BLOCK_SIZE} and match the cache")
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a [batch + 1] int32 tensor on the tokens' device")
    batch = cu_seqlens.numel() - 1
    cu = _int32_on("cu_seqlens", cu_seqlens, device, batch + 1)
    ctx = _int32_on("context_lens", context_lens, device, batch)
    shape = block_table.shape if isinstance(block_table, torch.Tensor) else ()
    if len(shape) != 2 or block_table.device != device or shape[0] < batch or shape[1] == 0:
        raise ValueError("block_table must be [>= batch, max_blocks_per_seq] on the tokens' device")
    if block_table.dtype != torch.int32:
        block_table = block_table.to(torch.int32)
    return batch, cu, ctx, block_table


def _chunk_args(q, k_cache, v_cache, block_table, block_size, cu_seqlens, context_lens, sm_scale,
                alibi_slopes, prefix_lens, scales=None):
    """Checks shared by the functions over packed new tokens and a paged cache (of 8-bit codes, if the
    function takes `scales`); returns the tensors as the library takes them."""
    _check_rows("q", q)
    if q.dim() != 3 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be [total_tokens, num_q_heads, {HEAD_DIM}]")
    shape = k_cache.shape if isinstance(k_cache, torch.Tensor) else None
    if scales is not None:
        _check_pages(k_cache, v_cache, *scales, q)
    else:
        _check_cache("k_cache", k_cache, q, shape)
        if v_cache is not None:
            _check_cache("v_cache", v_cache, q, shape)
    if q.shape[1] == 0 or q.shape[1] % shape[2] != 0:
        raise ValueError(f"num_q_heads {q.shape[1]} not a multiple of k/v heads {shape[2]}")
    device = q.device
    batch, cu, ctx, bt = _batch_args(device, block_table, block_size, k_cache, cu_seqlens,
                                     context_lens)
    prefix = None if prefix_lens is None else _int32_on("prefix_lens", prefix_lens, device, batch)
    slopes = None
    if alibi_slopes is not None:
        if (not isinstance(alibi_slopes, torch.Tensor) or alibi_slopes.device != device
                or alibi_slopes.shape != (q.shape[1],)):
            raise ValueError("alibi_slopes must be a [num_q_heads] float32 tensor on q's device")
        slopes = alibi_slopes.to(torch.float32).contiguous()
    scale = HEAD_DIM ** -0.5 if sm_scale is None else float(sm_scale)
    return batch, cu, ctx, prefix, bt, slopes, scale


def _ptr(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=4096)
def _chunk_workspace(device_index: int, total: int, num_q_heads: int, num_kv_heads: int) -> int:
    return int(_lib.load().fi_paged_chunk_workspace_size(total, num_q_heads, num_kv_heads))


@functools.lru_cache(maxsize=64)
def _mass_workspace(device_index: int) -> int:
    return int(_lib.load().fi_attention_mass_workspace_size())


def paged_chunk_workspace_bytes(total_tokens: int, num_q_heads: int, num_kv_heads: int) -> int:
    """Workspace bytes ``paged_chunk_attention`` needs for these sizes (current device)."""
    return int(_lib.load().fi_paged_chunk_workspace_size(total_tokens, num_q_heads, num_kv_heads))


def paged_chunk_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          block_table: torch.Tensor, block_size: int, cu_seqlens: torch.Tensor,
                          context_lens: torch.Tensor, sm_scale: float = None, *,
                          softcap: float = 0.0, alibi_slopes: torch.Tensor = None,
                          window: int = 0, prefix_lens: torch.Tensor = None,
                          return_lse: bool = False, out: torch.Tensor = None,
                          workspace: torch.Tensor = None):
    """Attention of new tokens over the paged cache that holds them and what came before:
    chunked prefill, verification of drafted tokens, single tokens, or a batch of all three.

    q: [total_tokens, num_q_heads, 128] fp16 or bf16, packed: sequence b owns rows
    [cu_seqlens[b], cu_seqlens[b+1]). k_cache, v_cache: [num_blocks, 64, num_kv_heads, 128] of
    q's type, already holding the new tokens' K and V; block_table: [>= batch, max_blocks].
    context_lens[b] counts the cached tokens with the new ones, so new token i of sequence b has
    position ``context_lens[b] - n_b + i``.

    Token p sees key j when j <= p (and j > p - window, if ``window``), or j < prefix_lens[b];
    never past context_lens[b]. Scores are ``q.k * sm_scale``, capped as ``softcap * tanh(x /
    softcap)`` if ``softcap``, less ``alibi_slopes[head] * |p - j|`` if given (fp32 [num_q_heads]).
    A token that sees nothing gives zeros and an lse of -inf. Slots past context_lens[b] may hold
    anything; V before them has to be finite, seen or not (hidden keys count with weight 0). A key
    whose score is -inf has weight 0; a NaN or +inf score makes NaN of the rows that see it. Pages with
    an invalid block-table entry are skipped and lengths that do not fit are cut, which only device
    checks (``FAST_INFER_B200_CHECK=1``) report, with a RuntimeError.

    Returns o like q (written to ``out`` if given; rows outside every sequence are not written),
    and with ``return_lse`` also lse: fp32 [total_tokens, num_q_heads], the natural log of the sum
    of exp(score). ``workspace``: uint8, at least ``paged_chunk_workspace_bytes`` bytes; calls that
    may run at the same time need one each (the default allocates per call).
    """
    batch, cu, ctx, prefix, bt, slopes, scale = _chunk_args(
        q, k_cache, v_cache, block_table, block_size, cu_seqlens, context_lens, sm_scale,
        alibi_slopes, prefix_lens)
    total, num_q_heads, _ = q.shape
    num_blocks, _, num_kv_heads, _ = k_cache.shape
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must be shaped and typed like q")
    lse = torch.empty(total, num_q_heads, dtype=torch.float32, device=q.device) \
        if return_lse else None
    if batch > 0 and total > 0:
        qx = q if _tma_ready(q) else q.clone(memory_format=torch.contiguous_format)
        ox = out if _tma_ready(out) else out.clone(memory_format=torch.contiguous_format)
        lib = _lib.load()
        with with_device(q.device):
            if workspace is None:
                workspace = torch.empty(
                    _chunk_workspace(q.device.index, total, num_q_heads, num_kv_heads),
                    dtype=torch.uint8, device=q.device)
            elif workspace.device != q.device or not workspace.is_contiguous():
                raise ValueError("workspace must be contiguous on q's device")
            err = error_word(q.device)
            st = lib.fi_paged_chunk(
                qx.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), ox.data_ptr(), _ptr(lse),
                bt.data_ptr(), cu.data_ptr(), ctx.data_ptr(), _ptr(prefix), _ptr(slopes), batch,
                total, num_q_heads, num_kv_heads, HEAD_DIM, num_blocks, block_size, bt.shape[1],
                _lib.strides(*qx.stride()), _lib.strides(*k_cache.stride()),
                _lib.strides(*v_cache.stride()), _lib.strides(*ox.stride()),
                _lib.strides(*bt.stride()), scale, float(softcap), int(window), _DTYPES[q.dtype],
                workspace.data_ptr(), workspace.numel() * workspace.element_size(), _ptr(err),
                stream_of(q.device))
            _lib.check(st, "paged_chunk_attention")
            device_errors(err, "paged_chunk_attention")
        if ox is not out:
            out.copy_(ox)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=4096)
def _tree_workspace(device_index: int, total: int, num_q_heads: int, num_kv_heads: int) -> int:
    return int(_lib.load().fi_paged_tree_workspace_size(total, num_q_heads, num_kv_heads))


def paged_tree_workspace_bytes(total_tokens: int, num_q_heads: int, num_kv_heads: int) -> int:
    """Workspace bytes ``paged_tree_attention`` needs for these sizes (current device)."""
    return int(_lib.load().fi_paged_tree_workspace_size(total_tokens, num_q_heads, num_kv_heads))


def paged_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         block_table: torch.Tensor, block_size: int, cu_seqlens: torch.Tensor,
                         context_lens: torch.Tensor, sm_scale: float = None, *,
                         tree_mask: torch.Tensor = None, depths: torch.Tensor = None,
                         k_scale: torch.Tensor = None, v_scale: torch.Tensor = None,
                         softcap: float = 0.0, window: int = 0, return_lse: bool = False,
                         out: torch.Tensor = None, workspace: torch.Tensor = None):
    """Attention of trees of drafted tokens over the paged cache that holds them and what came
    before, 16-bit or of 8-bit codes; without a tree, of single tokens, chains and prompts' chunks.

    q, block_table, cu_seqlens, context_lens, sm_scale, softcap, out, workspace: as in
    ``paged_chunk_attention`` (new token i of sequence b lies in slot ``context_lens[b] - n_b + i``).
    k_cache, v_cache: [num_blocks, 64, num_kv_heads, 128] of q's type; or codes, int8 or
    float8_e4m3fn, with k_scale, v_scale (fp32 [num_blocks, num_kv_heads, 64]), as
    ``rope_axes_store`` writes them: a row stands for code * scale.

    tree_mask: int32 [total_tokens, words] (``kernels.drafting.draft_tree``): new token i sees new
    token j of its sequence where bit j % 32 of word j // 32 is set, and every token cached before
    them. With ``window``, a token of position ``context_lens[b] - n_b + depths[i]`` (depths: int32
    [total_tokens], from ``draft_tree`` too) sees of those before the new ones only what is less than
    ``window`` behind it; among the new ones the mask alone decides (give ``draft_tree`` the window).
    Without tree_mask the new tokens are a chain: ``paged_chunk_attention``, which this equals for
    16-bit caches.

    A token that sees nothing gives zeros and an lse of -inf. Slots past context_lens[b] may hold
    anything; V (and its scale) before them has to be finite, seen or not. A key whose score is -inf
    has weight 0; a NaN or +inf score makes NaN of the rows that see it. Pages with an invalid
    block-table entry are skipped and lengths that do not fit are cut, which only device checks
    (``FAST_INFER_B200_CHECK=1``) report, with a RuntimeError.

    Returns o like q (rows outside every sequence are not written), and with ``return_lse`` also lse:
    fp32 [total_tokens, num_q_heads]. ``workspace``: uint8, at least ``paged_tree_workspace_bytes``.
    """
    batch, cu, ctx, _, bt, _, scale = _chunk_args(
        q, k_cache, v_cache, block_table, block_size, cu_seqlens, context_lens, sm_scale, None, None,
        (k_scale, v_scale))
    total, num_q_heads, _ = q.shape
    num_blocks, _, num_kv_heads, _ = k_cache.shape
    device = q.device
    words = 0
    if tree_mask is not None:
        if (not isinstance(tree_mask, torch.Tensor) or tree_mask.dim() != 2
                or tree_mask.dtype != torch.int32 or tree_mask.device != device
                or tree_mask.shape[0] != total or tree_mask.shape[1] == 0):
            raise ValueError("tree_mask must be an int32 tensor [total_tokens, words] on q's device")
        if window and depths is None:
            raise ValueError("a window over a tree needs depths")
        tree_mask, words = tree_mask.contiguous(), tree_mask.shape[1]
    if depths is not None:
        depths = _int32_on("depths", depths, device, total)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device:
        raise ValueError("out must be shaped and typed like q")
    lse = torch.empty(total, num_q_heads, dtype=torch.float32, device=device) \
        if return_lse else None
    if batch > 0 and total > 0:
        qx = q if _tma_ready(q) else q.clone(memory_format=torch.contiguous_format)
        ox = out if _tma_ready(out) else out.clone(memory_format=torch.contiguous_format)
        lib = _lib.load()
        with with_device(device):
            if workspace is None:
                workspace = torch.empty(
                    _tree_workspace(device.index, total, num_q_heads, num_kv_heads),
                    dtype=torch.uint8, device=device)
            elif workspace.device != device or not workspace.is_contiguous():
                raise ValueError("workspace must be contiguous on q's device")
            err = error_word(device)
            st = lib.fi_paged_tree(
                qx.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _ptr(k_scale), _ptr(v_scale),
                ox.data_ptr(), _ptr(lse), bt.data_ptr(), cu.data_ptr(), ctx.data_ptr(),
                _ptr(tree_mask), _ptr(depths), words, batch, total, num_q_heads, num_kv_heads,
                HEAD_DIM, num_blocks, block_size, bt.shape[1], _lib.strides(*qx.stride()),
                _lib.strides(*k_cache.stride()), _lib.strides(*v_cache.stride()),
                None if k_scale is None else _lib.strides(*k_scale.stride()),
                None if v_scale is None else _lib.strides(*v_scale.stride()),
                _lib.strides(*ox.stride()), _lib.strides(*bt.stride()), scale, float(softcap),
                int(window), _DTYPES[q.dtype], POOL_DTYPES[k_cache.dtype], workspace.data_ptr(),
                workspace.numel() * workspace.element_size(), _ptr(err), stream_of(device))
            _lib.check(st, "paged_tree_attention")
            device_errors(err, "paged_tree_attention")
        if ox is not out:
            out.copy_(ox)
    return (out, lse) if return_lse else out


def attention_mass(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor,
                   block_size: int, cu_seqlens: torch.Tensor, context_lens: torch.Tensor,
                   lse: torch.Tensor, sm_scale: float = None, *, softcap: float = 0.0,
                   alibi_slopes: torch.Tensor = None, window: int = 0,
                   prefix_lens: torch.Tensor = None, mass: torch.Tensor = None,
                   workspace: torch.Tensor = None) -> torch.Tensor:
    """Attention weight that each cached token receives from the new tokens, per KV head.

    ``mass[b, hk, j]`` = sum of ``exp(score - lse)`` over sequence b's new tokens and the query
    heads of hk. Arguments and score form as in ``paged_chunk_attention``, whose ``lse`` this takes;
    pass the last tokens alone (with ``cu_seqlens`` to match) for the weight of a window of
    them. ``mass``: fp32 [batch, num_kv_heads, capacity] to add to and return (what cached
    tokens had before); without it, a new one of the block table's span, 0 where nothing sees. The
    weights of cached tokens past a ``mass`` that is shorter than a sequence are dropped, which only
    device checks (``FAST_INFER_B200_CHECK=1``) report, with a RuntimeError.
    ``workspace``: uint8, at least ``attention_mass_workspace_bytes`` bytes; calls that may run at
    the same time need one each (the default allocates per call).
    """
    if k_cache is None:
        raise TypeError("k_cache must be a torch.Tensor")
    batch, cu, ctx, prefix, bt, slopes, scale = _chunk_args(
        q, k_cache, None, block_table, block_size, cu_seqlens, context_lens, sm_scale,
        alibi_slopes, prefix_lens)
    total, num_q_heads, _ = q.shape
    num_blocks, _, num_kv_heads, _ = k_cache.shape
    if (not isinstance(lse, torch.Tensor) or lse.shape != (total, num_q_heads)
            or lse.dtype != torch.float32 or lse.device != q.device):
        raise ValueError("lse must be [total_tokens, num_q_heads] float32 on q's device")
    accumulate = mass is not None
    if mass is None:
        mass = torch.empty(batch, num_kv_heads, bt.shape[1] * BLOCK_SIZE, dtype=torch.float32,
                           device=q.device)
    elif (mass.dim() != 3 or mass.shape[:2] != (batch, num_kv_heads) or not mass.is_contiguous()
          or mass.dtype != torch.float32 or mass.device != q.device):
        raise ValueError("mass must be a contiguous [batch, num_kv_heads, capacity] float32 tensor "
                         "on q's device")
    if mass.numel() == 0:
        return mass
    qx = q if _tma_ready(q) else q.clone(memory_format=torch.contiguous_format)
    lse = lse.contiguous()
    lib = _lib.load()
    with with_device(q.device):
        if workspace is None:
            workspace = torch.empty(_mass_workspace(q.device.index), dtype=torch.uint8,
                                    device=q.device)
        elif workspace.device != q.device or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous on q's device")
        err = error_word(q.device)
        st = lib.fi_attention_mass(
            qx.data_ptr(), k_cache.data_ptr(), lse.data_ptr(), mass.data_ptr(), bt.data_ptr(),
            cu.data_ptr(), ctx.data_ptr(), _ptr(prefix), _ptr(slopes), batch, total, num_q_heads,
            num_kv_heads, HEAD_DIM, num_blocks, block_size, bt.shape[1],
            _lib.strides(*qx.stride()), _lib.strides(*k_cache.stride()),
            _lib.strides(*bt.stride()), mass.shape[2], int(accumulate), scale, float(softcap),
            int(window), _DTYPES[q.dtype], workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), _ptr(err), stream_of(q.device))
        _lib.check(st, "attention_mass")
        device_errors(err, "attention_mass")
    return mass


def attention_mass_workspace_bytes() -> int:
    """Workspace bytes ``attention_mass`` needs (current device)."""
    return int(_lib.load().fi_attention_mass_workspace_size())
