"""Rotary positions with several axes and the slot write, against the definition in 64 bits."""

import pytest
import torch

from oracle.chunk_oracle import rope_axes

pytestmark = pytest.mark.gpu
PAGE, D = 64, 128


def tables(rows=500):
    freq = 1.0 / (10000.0 ** (torch.arange(0, D, 2).double() / D))
    ang = torch.outer(torch.arange(rows).double(), freq)
    ang = torch.cat([ang, ang], -1)
    return ang.cos().float(), ang.sin().float()


def make(seqs, nq, nkv, axes, dtype, seed=0, rows=500):
    g = torch.Generator().manual_seed(seed)
    total = sum(n for n, _ in seqs)
    pages = [(max(c, 0) + PAGE - 1) // PAGE for _, c in seqs]
    nb = sum(pages) + 2
    order = torch.randperm(nb, generator=g).int()
    table = torch.full((len(seqs), max(pages + [0]) + 1), -1, dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    qkv = torch.randn(total, (nq + 2 * nkv) * D, generator=g).to(dtype)
    pos = torch.randint(0, rows, (axes, total), generator=g).int()
    cu = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).int()
    return qkv, pos, table, cu, torch.tensor([c for _, c in seqs]).int(), nb


def check(case, sections, nq, nkv, dtype, dev, q, kc, vc, fill):
    """A value is products and a sum in fp32 (2^-22 of |x cos| + |y sin| together), rounded once
    (half a step); v is copied."""
    qkv, pos, table, cu, ctx, nb = case
    cos, sin = tables()
    x = qkv.view(-1, nq + 2 * nkv, D)
    ref = rope_axes(x[:, :nq + nkv], pos, sections, cos, sin)
    u = torch.finfo(dtype).eps / 2
    tol = u * ref.abs() + 2.0 ** -21 * x[:, :nq + nkv].abs().amax(-1, keepdim=True).double() + \
        (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((q.cpu().double() - ref[:, :nq]).abs() <= tol[:, :nq]).all()
    want_k = torch.zeros(nb, PAGE, nkv, D, dtype=torch.float64)
    owner = torch.zeros(nb, PAGE, dtype=torch.bool)
    for b in range(len(ctx)):
        for t in range(int(cu[b]), int(cu[b + 1])):
            slot = int(ctx[b]) - (int(cu[b + 1]) - t)
            page = int(table[b, slot // PAGE])
            owner[page, slot % PAGE] = True
            want_k[page, slot % PAGE] = ref[t, nq:]
            kt = kc[page, slot % PAGE].cpu().double()
            assert ((kt - ref[t, nq:]).abs() <= tol[t, nq:]).all()
            assert torch.equal(vc[page, slot % PAGE].cpu(), x[t, nq + nkv:])
    assert (kc.cpu()[~owner] == fill).all() and (vc.cpu()[~owner] == fill).all()


def run(case, sections, nq, nkv, dtype, dev, fill=7.0):
    from fast_infer_b200.kernels.rope import rope_axes_store
    qkv, pos, table, cu, ctx, nb = case
    kc = torch.full((nb, PAGE, nkv, D), fill, dtype=dtype, device=dev)
    vc = torch.full_like(kc, fill)
    cos, sin = (t.to(dev) for t in tables())
    q = rope_axes_store(qkv.to(dev), nq, cos, sin, pos.to(dev), sections, kc, vc, table.to(dev), PAGE,
                        cu.to(dev), ctx.to(dev))
    check(case, sections, nq, nkv, dtype, dev, q, kc, vc, fill)


SEQS = {"one": [(1, 1)], "decode": [(1, c) for c in (5, 64, 65, 129, 300)],
        "mixed": [(70, 70), (0, 33), (1, 65), (130, 200), (3, 128)]}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sections", [(64,), (16, 24, 24), (1, 63), (0, 5, 59, 0), (10, 20, 30, 4)])
@pytest.mark.parametrize("name", list(SEQS))
def test_axes(cuda_device, device_checks, name, sections, dtype):
    run(make(SEQS[name], 6, 2, len(sections), dtype), sections, 6, 2, dtype, cuda_device)


@pytest.mark.parametrize("nq,nkv", [(1, 1), (24, 8), (7, 1), (5, 5)])
def test_heads(cuda_device, device_checks, nq, nkv):
    run(make(SEQS["mixed"], nq, nkv, 3, torch.float16), (16, 24, 24), nq, nkv, torch.float16, cuda_device)


def test_agrees_with_rope_and_store(cuda_device, device_checks):
    """One axis whose position is the slot: rope_and_store's results within its extra fp16 roundings
    (two products and the cos / sin rows rounded as well: four half steps of the largest value)."""
    from fast_infer_b200.kernels.rope import rope_axes_store
    from fast_infer_b200.kv_cache import KVCache, rope_and_store
    B, S, nq, nkv = 2, 90, 6, 2
    cos, sin = (t.to(cuda_device) for t in tables())
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(B, S, (nq + 2 * nkv) * D, generator=g).half().to(cuda_device)
    a, b = (KVCache(1, nkv, D, 256, PAGE, cuda_device, num_blocks=8) for _ in range(2))
    cu, ctx = a.extend([S, S])
    b.extend([S, S])
    pos = torch.arange(S, device=cuda_device).repeat(B)[None].int()
    q1 = rope_axes_store(qkv.view(B * S, -1), nq, cos, sin, pos, (64,), a.k[0], a.v[0], a.block_table,
                         PAGE, cu, ctx)
    q2 = rope_and_store(b, 0, qkv, nq, cos, sin, 0).view(B * S, nq, D)
    tol = 4 * 2.0 ** -11 * 2 * float(qkv.abs().max())
    assert (q1.float() - q2.float()).abs().max() <= tol
    assert (a.k.float() - b.k.float()).abs().max() <= tol and torch.equal(a.v, b.v)


def test_rows_outside_stay_and_bad_places_are_reported(cuda_device):
    from fast_infer_b200._runtime import device_checks as checks
    from fast_infer_b200.kernels.rope import rope_axes_store
    qkv, pos, table, cu, ctx, nb = make([(5, 70), (9, 9)], 6, 2, 1, torch.float16)
    cos, sin = (t.to(cuda_device) for t in tables())

    def call(pos=pos, table=table, cu=cu, ctx=ctx):
        kc = torch.full((nb, PAGE, 2, D), 7.0, dtype=torch.float16, device=cuda_device)
        vc = torch.full_like(kc, 7.0)
        x = torch.cat([qkv, qkv[:6]]).to(cuda_device)
        p = torch.cat([pos, torch.full((1, 6), -9).int()], 1).to(cuda_device)
        out = torch.full((20, 6, D), 7.0, dtype=torch.float16, device=cuda_device)
        rope_axes_store(x, 6, cos, sin, p, (64,), kc, vc, table.to(cuda_device), PAGE,
                        cu.to(cuda_device), ctx.to(cuda_device), q_out=out)
        return out, kc, vc
    with checks(True):
        out, _, _ = call()
        assert (out[14:] == 7.0).all() and not (out[:14] == 7.0).all(-1).any()
        for kw, match in ((dict(pos=pos + 496), "context length"), (dict(table=table * 0 - 1), "page pool"),
                          (dict(table=table * 0 + nb), "page pool"), (dict(ctx=ctx - 8), "page pool"),
                          (dict(ctx=ctx + 4000), "page pool"),
                          (dict(cu=torch.tensor([0, 14, 5]).int()), "context length")):
            with pytest.raises(RuntimeError, match=match):
                call(**kw)
    out, kc, vc = call(table=table * 0 - 1)  # q comes back all the same, the cache is not touched
    assert not (out[:14] == 7.0).all(-1).any() and (kc == 7.0).all() and (vc == 7.0).all()
