"""Strides of dimensions of size 1 are never stepped over, so any will do: one token of a row-padded buffer, one head of a
padded pool, one layer, one page; results are those of dense tensors, bit for bit."""

import pytest
import torch

from tests.test_gpu_paged_chunk import make
from tests.test_gpu_rope_axes import tables

pytestmark = pytest.mark.gpu
PAGE, D = 64, 128


def odd(t):
    """t's values with an odd stride in every dimension of size 1 (and a base as aligned as t's)."""
    strides, step = [1], D
    for size in reversed(t.shape[:-1]):
        strides.insert(0, step + 1 if size == 1 else step)
        step *= size
    buf = torch.zeros(step + 64, dtype=t.dtype, device=t.device)
    x = buf.as_strided(t.shape, strides)
    x.copy_(t)
    assert any(s % 8 for s in x.stride()[:-1])
    return x


@pytest.mark.parametrize("hq,hk,seqs", [(6, 2, [(1, 200)]), (1, 1, [(1, 60)]), (1, 1, [(40, 150)]), (40, 1, [(1, 300)])])
def test_attention_and_mass(cuda_device, device_checks, hq, hk, seqs):
    from fast_infer_b200.kernels.attention import attention_mass, paged_chunk_attention
    q, k, v, table, cu, ctx = (t.to(cuda_device) for t in make(seqs, hq, hk, torch.float16, garbage=0.0, spare=0))
    want, lse = paged_chunk_attention(q, k, v, table, PAGE, cu, ctx, return_lse=True)
    out = odd(torch.zeros_like(q))
    if hk == 1:
        k, v = odd(k), odd(v)
    got, lse2 = paged_chunk_attention(odd(q), k, v, table, PAGE, cu, ctx, return_lse=True, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want) and torch.equal(lse2, lse)
    assert torch.equal(attention_mass(odd(q), k, table, PAGE, cu, ctx, lse),
                       attention_mass(q, k.contiguous(), table, PAGE, cu, ctx, lse))


@pytest.mark.parametrize("nq,nkv,total", [(6, 2, 1), (1, 1, 1), (1, 1, 40)])
def test_rope(cuda_device, device_checks, nq, nkv, total):
    from fast_infer_b200.kernels.rope import rope_axes_store
    cos, sin = (t.to(cuda_device) for t in tables())
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(total, (nq + 2 * nkv) * D, generator=g).half().to(cuda_device)
    pos = torch.randint(0, 500, (1, total), generator=g).int().to(cuda_device)
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device)
    cu = torch.tensor([0, total], dtype=torch.int32, device=cuda_device)
    ctx = cu[1:] + 5

    def call(x, kc, vc, out):
        q = rope_axes_store(x, nq, cos, sin, pos, (64,), kc, vc, table, PAGE, cu, ctx, q_out=out)
        return q, kc, vc
    pool = torch.zeros(1, PAGE, nkv, D, dtype=torch.float16, device=cuda_device)
    want = call(qkv, pool.clone(), pool.clone(), None)
    wide = torch.empty(total, qkv.shape[1] + 3, dtype=qkv.dtype, device=cuda_device)[:, :qkv.shape[1]]
    wide.copy_(qkv)  # (with more than one token it is copied: the rows are not aligned)
    out = odd(torch.zeros(total, nq, D, dtype=qkv.dtype, device=cuda_device))
    got = call(wide, odd(pool), odd(pool), out)
    assert got[0].data_ptr() == out.data_ptr() and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("layers,heads", [(1, 2), (2, 1), (1, 1)])
def test_evict(cuda_device, device_checks, layers, heads):
    from fast_infer_b200.kernels.eviction import evict_tokens
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(layers, 1, PAGE, heads, D, generator=g).half().to(cuda_device) for _ in range(2))
    mass = torch.rand(layers, 1, heads, PAGE, generator=g).to(cuda_device)
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([50], dtype=torch.int32, device=cuda_device)
    dense = (k.clone(), v.clone())
    want = evict_tokens(*dense, table, lens, mass, 20, recent=3, sinks=1)
    ko, vo = odd(k), odd(v)
    got = evict_tokens(ko, vo, table, lens, mass, 20, recent=3, sinks=1)
    assert all(torch.equal(a, b) for a, b in zip(got + (ko, vo), want + dense))
    to = (odd(torch.zeros_like(k)), odd(torch.zeros_like(v)), table.clone())
    got = evict_tokens(odd(k), odd(v), table, lens, mass, 20, recent=3, sinks=1, out=to)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(to[0][:, :, :20], dense[0][:, :, :20]) and torch.equal(to[1][:, :, :20], dense[1][:, :, :20])
