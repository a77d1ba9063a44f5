"""The whole loop of a server that drafts, over caches of every type: extend, draft_tree, rope_axes_store, paged_tree_attention,
sample_tokens, accept_drafts, KVCache.accept. After every step the cache has to hold exactly what a cache holds that was given
the accepted tokens alone, one after another (the same kernel wrote both: equal bits), and the next attention has to see it."""

import math

import numpy as np
import pytest
import torch

from fast_infer_b200.kernels.attention import paged_tree_attention
from fast_infer_b200.kernels.drafting import accept_drafts, draft_tree
from fast_infer_b200.kernels.rope import read_kv, rope_axes_store
from fast_infer_b200.kernels.sampling import sample_tokens
from fast_infer_b200.kv_cache import KVCache

pytestmark = pytest.mark.gpu
LAYERS, HQ, HK, VOCAB = 2, 6, 2, 5


@pytest.mark.parametrize("pool", [torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn])
def test_loop(cuda_device, device_checks, pool):
    dev = cuda_device
    coded = pool in (torch.int8, torch.float8_e4m3fn)
    dtype = torch.bfloat16 if pool == torch.bfloat16 else torch.float16
    rng = np.random.default_rng(3)
    g = torch.Generator(device=dev).manual_seed(3)
    cache, plain = (KVCache(LAYERS, HK, 128, 512, 64, dev, num_blocks=24, dtype=pool) for _ in range(2))
    freq = 1.0 / (10000.0 ** (torch.arange(0, 128, 2, device=dev).double() / 128))
    angle = torch.outer(torch.arange(600, device=dev).double(), freq)
    cos, sin = (torch.cat([f(angle), f(angle)], -1).float() for f in (torch.cos, torch.sin))

    def store(c, layer, qkv, pos, cu, ctx):
        scales = dict(k_scale=c.k_scale[layer], v_scale=c.v_scale[layer]) if coded else {}
        return rope_axes_store(qkv, HQ, cos, sin, pos[None], (64,), c.k[layer], c.v[layer], c.block_table, 64, cu, ctx, **scales)

    lengths = np.zeros(3, np.int64)
    for step in range(9):
        # prompts, trees of several shapes, a step where a sequence sits out, single tokens
        new = [(70, 3, 30), (20, 26, 5), (9, 0, 33), (1, 1, 1), (40, 12, 2), (1, 64, 7), (3, 3, 3), (25, 1, 0), (50, 8, 8)][step]
        par = []
        for n in new:
            i = np.arange(n)
            par.append(i - 1 if step == 0 else i - 1 - np.floor(rng.random(n) * np.minimum(i, 4)).astype(np.int64))
        parents = torch.from_numpy(np.concatenate(par).astype(np.int32)).to(dev)
        total = sum(new)
        cu, ctx = cache.extend(new)
        mask, depths = draft_tree(parents, cu, max(new))
        start = torch.repeat_interleave(torch.from_numpy(lengths).to(dev).int(), torch.tensor(new, device=dev))
        qkv = torch.randn(LAYERS, total, (HQ + 2 * HK) * 128, generator=g, device=dev).to(dtype)
        for layer in range(LAYERS):
            q = store(cache, layer, qkv[layer], start + depths, cu, ctx)
            o, lse = paged_tree_attention(q, cache.k[layer], cache.v[layer], cache.block_table, 64, cu, ctx, tree_mask=mask,
                                          k_scale=cache.k_scale[layer] if coded else None,
                                          v_scale=cache.v_scale[layer] if coded else None, return_lse=True)
            assert torch.isfinite(o).all() and torch.isfinite(lse).all()
        logits = (o.float().view(total, -1)[:, :VOCAB] * 5).to(torch.bfloat16)
        sampled = sample_tokens(logits, torch.rand(total, generator=g, device=dev), 0.7, top_k=4, top_p=0.95)
        assert ((sampled >= 0) & (sampled < VOCAB)).all()
        tokens = torch.randint(0, VOCAB, (total,), generator=g, device=dev, dtype=torch.int32)
        if step == 0:  # a prompt: every token stands
            tokens = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), sampled[:-1]])
        path, counts, follow = accept_drafts(tokens, sampled, parents, cu)
        kept = cache.accept(cu, ctx, path, counts)
        assert kept.tolist() == counts.tolist()
        if step == 0:
            assert kept.tolist() == list(new)
        # the accepted rows alone, into the other cache
        pick, p = [], path.tolist()
        at = 0
        for n, c in zip(new, kept):
            pick += [at + node for node in p[at:at + c]]
            at += n
        pick = torch.tensor(pick, dtype=torch.long, device=dev)
        cu2, ctx2 = plain.extend(kept)
        pos2 = torch.cat([torch.arange(l, l + c, device=dev) for l, c in zip(lengths, kept)]).int()
        for layer in range(LAYERS):
            store(plain, layer, qkv[layer][pick].contiguous(), pos2, cu2, ctx2)
        lengths += kept
        assert cache.seq_lens[:3].tolist() == lengths.tolist() == plain.seq_lens[:3].tolist()
        assert len(cache.free_blocks) == 24 - int(sum(-(-l // 64) for l in lengths))
        for layer in range(LAYERS):
            for b, l in enumerate(lengths):
                for a, c in ((cache.k, plain.k), (cache.v, plain.v)):
                    rows = [x[layer][y.block_table[b, :-(-l // 64)].long()].reshape(-1, HK, 128)[:l]
                            for x, y in ((a, cache), (c, plain))]
                    as_int = torch.int8 if coded else torch.int16
                    assert torch.equal(rows[0].view(as_int), rows[1].view(as_int))
        # a token after it all sees the same in both, read back and through the attention
        whole = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).to(dev)
        lens = torch.from_numpy(lengths.astype(np.int32)).to(dev)
        one = torch.arange(4, dtype=torch.int32, device=dev)
        probe = torch.randn(3, HQ, 128, generator=g, device=dev).to(dtype)
        seen = []
        for c in (cache, plain):
            scales = dict(k_scale=c.k_scale[1], v_scale=c.v_scale[1]) if coded else {}
            seen.append(paged_tree_attention(probe, c.k[1], c.v[1], c.block_table, 64, one, lens, **scales))
            if coded:
                seen += list(read_kv(c.k[1], c.v[1], c.k_scale[1], c.v_scale[1], c.block_table, 64, whole, lens,
                                     int(lengths.sum()), dtype=dtype))
        for a, b in zip(seen[:len(seen) // 2], seen[len(seen) // 2:]):
            assert torch.equal(a, b)


def test_accept_changes_nothing_when_it_refuses(cuda_device):
    dev = cuda_device
    cache = KVCache(1, HK, 128, 256, 64, dev, num_blocks=8)
    cache.k.copy_(torch.randn(cache.k.shape, device=dev))
    cache.v.copy_(torch.randn(cache.v.shape, device=dev))
    cache.extend([30, 60])
    cu, ctx = cache.extend([5, 9])
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    path = ints(0, 2, 4, -1, -1, 0, 3, 8, -1, -1, -1, -1, -1, -1)
    counts = ints(3, 3)
    was = cache.k.clone(), cache.v.clone(), cache.seq_lens.copy(), list(cache.free_blocks)
    for bad in ((cu, ctx, path, ints(6, 3)), (cu, ctx, path, ints(3, -1)), (cu, ctx - 1, path, counts), (cu + 1, ctx, path, counts),
                (cu, ctx, path[:10], counts), (cu, ctx, path, ints(3)), (cu[:2], ctx, path, counts)):
        with pytest.raises(ValueError):
            cache.accept(*bad)
        assert torch.equal(cache.k, was[0]) and torch.equal(cache.v, was[1])
        assert (cache.seq_lens == was[2]).all() and cache.free_blocks == was[3]
    assert cache.accept(cu, ctx, path, counts).tolist() == [3, 3] and cache.seq_lens.tolist() == [33, 63]
    assert len(cache.free_blocks) == len(was[3]) + 1
    with pytest.raises(ValueError):  # the same step twice
        cache.accept(cu, ctx, path, counts)


@pytest.mark.parametrize("pool", [torch.int8, torch.float8_e4m3fn])
def test_operators_of_16_bit_pages_refuse_codes(cuda_device, pool):
    """What does not take scales takes no codes."""
    from fast_infer_b200.kernels.attention import attention_mass, paged_attention, paged_chunk_attention
    from fast_infer_b200.kv_cache import rope_and_store, store_kv_decode, store_kv_prefill
    dev = cuda_device
    cache = KVCache(1, HK, 128, 256, 64, dev, num_blocks=8, dtype=pool)
    cu, ctx = cache.extend([5])
    q = torch.randn(5, HQ, 128, device=dev).half()
    lse = torch.zeros(5, HQ, device=dev)
    rows = torch.randn(1, 5, HK, 128, device=dev).half()
    tables = torch.ones(256, 128, device=dev)
    args = (cache.k[0], cache.v[0], cache.block_table, 64)
    with pytest.raises((TypeError, ValueError)):
        paged_chunk_attention(q, *args, cu, ctx)
    with pytest.raises((TypeError, ValueError)):
        paged_tree_attention(q, *args, cu, ctx)
    with pytest.raises((TypeError, ValueError)):
        paged_attention(q[:1], *args, 5)
    with pytest.raises((TypeError, ValueError)):
        attention_mass(q, cache.k[0], cache.block_table, 64, cu, ctx, lse)
    with pytest.raises((TypeError, ValueError)):
        cache.evict(torch.zeros(1, 1, HK, 256, device=dev), 2)
    with pytest.raises((TypeError, ValueError)):
        store_kv_prefill(cache, 0, rows, rows)
    with pytest.raises((TypeError, ValueError)):
        store_kv_decode(cache, 0, rows[:, 0], rows[:, 0], 6)
    with pytest.raises((TypeError, ValueError)):
        rope_and_store(cache, 0, torch.randn(1, 1, (HQ + 2 * HK) * 128, device=dev).half(), HQ, tables, tables, 0)
    assert (cache.k.view(torch.int8) == 0).all() and (cache.v.view(torch.int8) == 0).all()
