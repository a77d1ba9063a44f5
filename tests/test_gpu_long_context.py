"""A long context served in chunks over a bounded cache, the operators as they follow one another:
rotary positions and the slot write, attention over the cache, the weights each token received, and
eviction when a sequence outgrows its budget; every step against the same loop in 64 bits on what the
cache holds."""

import pytest
import torch

from oracle.chunk_oracle import chunk, evict_keep, mass as mass_oracle, rope_axes
from tests.test_gpu_paged_chunk import check as check_attention
from tests.test_gpu_rope_axes import tables

pytestmark = pytest.mark.gpu
PAGE, D = 64, 128


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_chunks_attention_weights_eviction(cuda_device, device_checks, dtype):
    from fast_infer_b200.kernels.attention import attention_mass, paged_chunk_attention
    from fast_infer_b200.kernels.rope import rope_axes_store
    from fast_infer_b200.kv_cache import KVCache
    nq, nkv, layers, budget = 6, 2, 2, 96
    cos, sin = tables()
    cosd, sind = cos.to(cuda_device), sin.to(cuda_device)
    cache = KVCache(layers, nkv, D, 512, PAGE, cuda_device, num_blocks=12, dtype=dtype)
    weights = torch.zeros(layers, 3, nkv, 512, device=cuda_device)
    seen = torch.zeros(3, dtype=torch.int64)  # positions of every sequence so far
    g = torch.Generator().manual_seed(11)
    sections = (16, 24, 24)
    for new in ([100, 40, 1], [60, 0, 80], [1, 1, 1], [70, 33, 20], [1, 1, 1]):
        cu, ctx = cache.extend(new)
        place = torch.cat([seen[b] + torch.arange(n) for b, n in enumerate(new)])
        pos = torch.stack([place, place // 2, place % 7]).int()
        seen += torch.tensor(new)
        for layer in range(layers):
            qkv = torch.randn(sum(new), (nq + 2 * nkv) * D, generator=g).to(dtype)
            kc, vc = cache.k[layer], cache.v[layer]
            q = rope_axes_store(qkv.to(cuda_device), nq, cosd, sind, pos.to(cuda_device), sections, kc, vc,
                                cache.block_table, PAGE, cu, ctx)
            x = qkv.view(-1, nq + 2 * nkv, D)
            ref = rope_axes(x[:, :nq], pos, sections, cos, sin)
            assert ((q.cpu().double() - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() + 1e-5).all()
            o, lse = paged_chunk_attention(q, kc, vc, cache.block_table, PAGE, cu, ctx, softcap=30.0,
                                           return_lse=True)
            held = (q.cpu(), kc.cpu(), vc.cpu(), cache.block_table.cpu(), cu.cpu(), ctx.cpu())
            check_attention(o, lse, chunk(*held, softcap=30.0), dtype)
            was = weights[layer].cpu().double()
            attention_mass(q, kc, cache.block_table, PAGE, cu, ctx, lse, softcap=30.0, mass=weights[layer])
            add = mass_oracle(held[0], held[1], *held[3:], lse.cpu(), softcap=30.0)
            n = min(add.shape[2], 512)
            want = was.clone()
            want[..., :n] += add[..., :n]
            assert ((weights[layer].cpu().double() - want).abs() <= want * 2.0 ** -15).all()
        before = (cache.k.cpu(), cache.v.cpu(), cache.block_table.cpu(), weights.cpu(), list(cache.seq_lens))
        kept = cache.evict(weights, budget, recent=16, sinks=2).cpu()
        for layer in range(layers):
            for b in range(3):
                for h in range(nkv):
                    idx = evict_keep(before[3][layer, b, h, :before[4][b]].tolist(), budget, 16, 2)
                    assert kept[layer, b, h, :len(idx)].tolist() == idx
                    j, r = torch.tensor(idx).long(), torch.arange(len(idx))
                    for old, now in ((before[0], cache.k), (before[1], cache.v)):
                        a = old[layer, before[2][b, j // PAGE].long(), j % PAGE, h]
                        c = now.cpu()[layer, cache.block_table.cpu()[b, r // PAGE].long(), r % PAGE, h]
                        assert torch.equal(a, c)
    assert list(cache.seq_lens) == [96, 40 + 0 + 1 + 33 + 1, 96]


def test_two_streams_at_once(cuda_device):
    """Two batches in flight on two streams, each with its own buffers, give what they give alone."""
    from fast_infer_b200.kernels.attention import attention_mass, paged_chunk_attention
    from tests.test_gpu_paged_chunk import make
    batches = [[t.to(cuda_device) for t in make([(200, 900), (1, 700)], 6, 2, torch.float16, s)]
               for s in (1, 2)]

    def call(b):
        o, lse = paged_chunk_attention(*b[:4], PAGE, *b[4:], return_lse=True)
        return o, lse, attention_mass(b[0], b[1], b[3], PAGE, b[4], b[5], lse)
    want = [call(b) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    for _ in range(5):
        got = []
        for s, b in zip(streams, batches):
            with torch.cuda.stream(s):
                got.append(call(b))
        torch.cuda.synchronize()
        for w, x in zip(want, got):
            assert all(torch.equal(i, j) for i, j in zip(w, x))
