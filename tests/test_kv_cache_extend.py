"""KVCache.extend that raises leaves the cache as it was, its batch and block table among the rest."""

import numpy as np
import pytest
import torch

from fast_infer_b200.kv_cache import KVCache


@pytest.mark.parametrize("n_new,match", [([10, 0, 300], "table full"), ([0, 100, 250], "out of memory"),
                                         ([1, 2, -1], "negative")])
def test_extend_that_raises_does_not_grow_the_batch(n_new, match):
    cache = KVCache(1, 2, 128, 256, 64, torch.device("cpu"), num_blocks=5)
    cache.extend([70, 64])
    table, rows, free, lens = (cache.block_table, cache.block_table.clone(), list(cache.free_blocks),
                               cache.seq_lens.copy())
    with pytest.raises((RuntimeError, ValueError), match=match):
        cache.extend(n_new)
    assert cache.block_table is table and torch.equal(table, rows) and cache._bt.shape == (2, 4)
    assert cache.free_blocks == free and np.array_equal(cache.seq_lens, lens)
    cu, ctx = cache.extend([1, 0, 100])  # and one that fits grows it
    assert cu.tolist() == [0, 1, 1, 101] and ctx.tolist() == [71, 64, 100]
    assert cache.block_table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [3, 4, -1, -1]]


def test_evict_refuses_pages_whose_tokens_it_does_not_know():
    """Tokens written by store / write_tokens into pages of alloc_block have no length: all their pages would go."""
    cache = KVCache(1, 2, 128, 256, 64, torch.device("cpu"), num_blocks=5)
    cache.alloc_block(0)
    with pytest.raises(ValueError, match="per-sequence"):
        cache.evict(torch.zeros(1, 1, 2, 256), 8)
    assert cache.free_blocks == [1, 2, 3, 4] and cache._bt[0, 0] == 0
