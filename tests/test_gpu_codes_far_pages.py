"""A pool of codes of more than 2^31 bytes: pages at its end are written, read, attended to and moved as those at its start."""

import pytest
import torch

from fast_infer_b200.kernels.attention import paged_tree_attention
from fast_infer_b200.kernels.drafting import keep_accepted
from fast_infer_b200.kernels.rope import read_kv, rope_axes_store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[3, 2], [70, 1]])  # (few rows alone, and both kernels)
def test_pages_past_32_bits(cuda_device, device_checks, new):
    dev, nq, nkv = cuda_device, 24, 8
    total, past = sum(new), [130, 500]
    pages = [-(-(p + n) // 64) for p, n in zip(past, new)]
    g = torch.Generator(device=dev).manual_seed(3)
    cu = torch.tensor([0, new[0], total], dtype=torch.int32, device=dev)
    ctx = torch.tensor([p + n for p, n in zip(past, new)], dtype=torch.int32, device=dev)
    before = torch.randn(sum(past), (nq + 2 * nkv) * 128, generator=g, device=dev).half()
    qkv = torch.randn(total, (nq + 2 * nkv) * 128, generator=g, device=dev).half()
    table = torch.ones(8, 128, device=dev), torch.zeros(8, 128, device=dev)  # (no rotation)
    path = torch.cat([torch.tensor([0] + [n - 1] * (n > 1) + [-1] * (n - 2), dtype=torch.int32) for n in new]).to(dev)
    counts = torch.tensor([min(n, 2) for n in new], dtype=torch.int32, device=dev)
    want = None
    for nb in (sum(pages) + 1, 34000):  # 34000 pages of 64 x 8 x 128 codes are 2.2 GB
        first = nb - sum(pages)
        bt = torch.full((2, max(pages)), -1, dtype=torch.int32, device=dev)
        bt[0, :pages[0]] = torch.arange(first, first + pages[0])
        bt[1, :pages[1]] = torch.arange(first + pages[0], nb)
        k, v = (torch.empty(1, nb, 64, nkv, 128, dtype=torch.int8, device=dev) for _ in "kv")
        ks, vs = (torch.zeros(1, nb, nkv, 64, device=dev) for _ in "kv")
        args = (k[0], v[0], bt, 64)
        scales = dict(k_scale=ks[0], v_scale=vs[0])
        old = torch.tensor([0, past[0], sum(past)], dtype=torch.int32, device=dev), torch.tensor(past, dtype=torch.int32, device=dev)
        pos = torch.zeros(1, sum(past), dtype=torch.int32, device=dev)
        rope_axes_store(before, nq, *table, pos, (64,), *args, *old, **scales)
        q = rope_axes_store(qkv, nq, *table, pos[:, :total], (64,), *args, cu, ctx, **scales)
        o, lse = paged_tree_attention(q, *args, cu, ctx, return_lse=True, **scales)
        keep_accepted(k, v, bt, 64, cu, ctx, path, counts, k_scale=ks, v_scale=vs)
        got = (o, lse) + read_kv(k[0], v[0], ks[0], vs[0], bt, 64, cu, ctx, total)
        assert torch.isfinite(o).all() and (got[2].abs().amax((1, 2)) > 0).all()
        if want is None:
            want = got
        else:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        del k, v, ks, vs
