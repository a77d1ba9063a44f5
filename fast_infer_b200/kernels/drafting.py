"""Drafted tokens (no counterpart in the reference, which decodes one token at a time): the shape of
draft trees, the acceptance of drafts, and the move of the accepted tokens' K and V.

A step of a server that drafts: ``draft_tree`` turns parents into ancestor masks and depths,
``kernels.attention.paged_tree_attention`` attends by the masks, ``kernels.sampling.sample_tokens``
samples a token after every node, ``accept_drafts`` walks the tree by them, and ``keep_accepted`` (or
``KVCache.accept``) leaves only the accepted tokens in the cache.
"""

from __future__ import annotations

import torch

from fast_infer_b200 import _lib
from fast_infer_b200._runtime import device_errors, error_word, stream_of, with_device
from fast_infer_b200.kernels.attention import (BLOCK_SIZE, HEAD_DIM, POOL_DTYPES, _check_scales,
                                               _int32_on, _ptr)


def _new_tokens(name: str, t: torch.Tensor):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (fast_infer_b200 has no CPU path)")
    if t.dim() != 1:
        raise ValueError(f"{name} must be a 1-D int32 tensor [total_tokens]")
    return t.device, t.numel(), _int32_on(name, t, t.device, t.numel())


def _batch_of(cu_seqlens, device):
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a [batch + 1] int32 tensor on the tokens' device")
    batch = cu_seqlens.numel() - 1
    return batch, _int32_on("cu_seqlens", cu_seqlens, device, batch + 1)


def draft_tree(parents: torch.Tensor, cu_seqlens: torch.Tensor, max_new: int, *,
               window: int = 0):
    """Ancestor masks and depths of draft trees.

    parents: int32 [total_tokens], packed by cu_seqlens; node i of a sequence is its new token i, and
    parents[i] (a number within the sequence, below i) its parent; any other value makes it a root.
    max_new (host int) bounds the new tokens of a sequence. Returns (mask, depths): int32
    [total_tokens, ceil(max_new / 32)], bit j % 32 of word j // 32 of row i set where node i sees
    node j (itself and its ancestors; with ``window`` the nearest ``window`` of them, itself among
    them), and int32 [total_tokens], the steps to the root: node i has position ``context_lens[b] -
    n_b + depths[i]``. Rows outside every sequence are not written. A sequence of more than
    32 * ceil(max_new / 32) new tokens loses the bits past the mask, which only device checks
    (``FAST_INFER_B200_CHECK=1``) report, with a RuntimeError.
    """
    device, total, parents = _new_tokens("parents", parents)
    batch, cu = _batch_of(cu_seqlens, device)
    max_new, window = int(max_new), int(window)
    if max_new < 1 or window < 0:
        raise ValueError(f"needs max_new >= 1 and window >= 0, got {max_new}, {window}")
    words = (max_new + 31) // 32
    mask = torch.empty(total, words, dtype=torch.int32, device=device)
    depths = torch.empty(total, dtype=torch.int32, device=device)
    if batch == 0 or total == 0:
        return mask, depths
    with with_device(device):
        err = error_word(device)
        st = _lib.load().fi_draft_tree(parents.data_ptr(), cu.data_ptr(), mask.data_ptr(),
                                       depths.data_ptr(), total, batch, words, window, _ptr(err),
                                       stream_of(device))
        _lib.check(st, "draft_tree")
        device_errors(err, "draft_tree")
    return mask, depths


def accept_drafts(tokens: torch.Tensor, sampled: torch.Tensor, parents: torch.Tensor,
                  cu_seqlens: torch.Tensor):
    """Which drafted tokens stand: from node 0 of each sequence (its last known token, always
    accepted) to the first child whose token is the one sampled after the node, until there is none.

    tokens, sampled, parents: int32 [total_tokens], packed by cu_seqlens: each node's token, the
    token that the model samples after it, and its parent (as in ``draft_tree``). Sampling after
    every node and accepting by equality leaves the distribution that of sampling token by token. A
    negative ``sampled`` (``sample_tokens`` gives -1 for a row that it cannot sample) ends the walk,
    whatever the drafts hold.
    Returns (path, counts, next_tokens): int32 [total_tokens], entry cu_seqlens[b] + d the number of
    the d-th accepted node, ascending, -1 past the last; int32 [batch], the nodes accepted; int32
    [batch], the token sampled after the last of them (-1 for a sequence without new tokens).
    """
    device, total, tokens = _new_tokens("tokens", tokens)
    sampled = _int32_on("sampled", sampled, device, total)
    parents = _int32_on("parents", parents, device, total)
    batch, cu = _batch_of(cu_seqlens, device)
    path = torch.empty(total, dtype=torch.int32, device=device)
    counts = torch.empty(batch, dtype=torch.int32, device=device)
    follow = torch.empty(batch, dtype=torch.int32, device=device)
    if batch == 0:
        return path, counts, follow
    with with_device(device):
        err = error_word(device)
        st = _lib.load().fi_accept_drafts(tokens.data_ptr(), sampled.data_ptr(),
                                          parents.data_ptr(), cu.data_ptr(), path.data_ptr(),
                                          counts.data_ptr(), follow.data_ptr(), total, batch,
                                          _ptr(err), stream_of(device))
        _lib.check(st, "accept_drafts")
        device_errors(err, "accept_drafts")
    return path, counts, follow


def keep_accepted(k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, block_size: int,
                  cu_seqlens: torch.Tensor, context_lens: torch.Tensor, path: torch.Tensor,
                  counts: torch.Tensor, *, k_scale: torch.Tensor = None,
                  v_scale: torch.Tensor = None) -> None:
    """Move the accepted tokens' K and V to consecutive slots, in place, all layers in one launch.

    k, v: [layers, num_blocks, 64, num_heads, 128] pools (``KVCache.k`` / ``.v``), fp16, bf16, int8 or
    float8_e4m3fn, the last two with k_scale, v_scale (``KVCache.k_scale`` / ``.v_scale``).
    block_table, cu_seqlens, context_lens: as in the attention call before; path, counts: from
    ``accept_drafts``. Afterwards sequence b holds ``context_lens[b] - n_b + counts[b]`` tokens; its
    slots past those are free. Pages must not be shared between sequences. A token whose page is
    missing is not moved, which only device checks (``FAST_INFER_B200_CHECK=1``) report, with a
    RuntimeError.
    """
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (fast_infer_b200 has no CPU path)")
        if t.dtype not in POOL_DTYPES:
            raise TypeError(f"{name} must be float16, bfloat16, int8 or float8_e4m3fn, got {t.dtype}")
        if t.dim() != 5 or t.shape[2] != BLOCK_SIZE or t.shape[4] != HEAD_DIM or 0 in t.shape[1:]:
            raise ValueError(f"{name} must be [layers, num_blocks, {BLOCK_SIZE}, num_heads, "
                             f"{HEAD_DIM}]")
    if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
        raise ValueError("k and v must have the same shape, type and device")
    if block_size != BLOCK_SIZE:
        raise ValueError(f"block_size must be {BLOCK_SIZE}")
    layers, num_blocks, _, heads, _ = k.shape
    device = k.device
    _check_scales(k, k_scale, v_scale, (layers, num_blocks, heads, BLOCK_SIZE))
    batch, cu = _batch_of(cu_seqlens, device)
    ctx = _int32_on("context_lens", context_lens, device, batch)
    counts = _int32_on("counts", counts, device, batch)
    if not isinstance(path, torch.Tensor) or path.dim() != 1:
        raise ValueError("path must be a 1-D int32 tensor [total_tokens] on the cache's device")
    total = path.numel()
    path = _int32_on("path", path, device, total)
    shape = block_table.shape if isinstance(block_table, torch.Tensor) else ()
    if len(shape) != 2 or shape[0] < batch or shape[1] == 0 or block_table.device != device:
        raise ValueError("block_table must be [>= batch, max_blocks] on the cache's device")
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    if layers == 0 or batch == 0 or total == 0:
        return
    with with_device(device):
        err = error_word(device)
        st = _lib.load().fi_keep_accepted(
            k.data_ptr(), v.data_ptr(), _ptr(k_scale), _ptr(v_scale), bt.data_ptr(), cu.data_ptr(),
            ctx.data_ptr(), path.data_ptr(), counts.data_ptr(), layers, batch, total, heads, HEAD_DIM,
            num_blocks, BLOCK_SIZE, bt.shape[1], _lib.strides(*k.stride()),
            _lib.strides(*v.stride()),
            None if k_scale is None else _lib.strides(*k_scale.stride()),
            None if v_scale is None else _lib.strides(*v_scale.stride()),
            _lib.strides(*bt.stride()), POOL_DTYPES[k.dtype], _ptr(err), stream_of(device))
        _lib.check(st, "keep_accepted")
        device_errors(err, "keep_accepted")
