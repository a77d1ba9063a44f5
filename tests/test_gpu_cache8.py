"""A cache of 8-bit codes: written by rope_axes_store, read back by read_kv.

Codes of values that go in as they are (v; k at position 0, whose rotation is the identity) are those of exact arithmetic,
ties included, so they have to be equal. A rotated k is off by 3 roundings of fp32 of at most sqrt(2) max|x| each before it is
quantised: in steps of a code (max|x| / 127) that is 3 * 2^-24 * 1.42 * 127 < 4e-5, beside half a step of the code itself."""

import math

import numpy as np
import pytest
import torch

from fast_infer_b200.kernels.rope import read_kv, rope_axes_store

pytestmark = pytest.mark.gpu
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def exact_codes(x, kind):
    """Codes (as values) and scales of rows x in 64 bits."""
    top_code = CODES[kind][1]
    top = x.double().abs().amax(-1, keepdim=True)
    z = x.double() * top_code / torch.where(top > 0, top, 1.0)
    if kind == "int8":
        step = torch.ones_like(z)
    else:
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(z / step) * step, (top / top_code)[..., 0], step


def tables(dev, rows=5000):
    freq = 1.0 / (10000.0 ** (torch.arange(0, 128, 2, device=dev).double() / 128))
    angle = torch.outer(torch.arange(rows, device=dev).double(), freq)
    angle = torch.cat([angle, angle], -1)
    return angle.cos().float(), angle.sin().float()


def batch(dev, new, past, seed=0):
    rng = np.random.default_rng(seed)
    ctx = np.array(new) + np.array(past)
    pages = -(-ctx // 64)
    nb = int(pages.sum()) + 2
    order, at = rng.permutation(nb), 0
    table = np.full((len(new), int(pages.max()) + 1), -1, np.int32)
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    slots = [(b, s) for b in range(len(new)) for s in range(past[b], past[b] + new[b])]
    where = (torch.tensor([int(table[b, s // 64]) for b, s in slots], dtype=torch.long, device=dev),
             torch.tensor([s % 64 for _, s in slots], dtype=torch.long, device=dev))
    return (torch.from_numpy(table).to(dev), torch.from_numpy(cu).to(dev),
            torch.from_numpy(ctx.astype(np.int32)).to(dev), nb, where)


def pools(dev, nb, hk, kind):
    k = torch.full((nb, 64, hk, 128), 3, device=dev).to(CODES[kind][0])
    ks = torch.full((nb, hk, 64), 7.0, device=dev)
    return k, k.clone(), ks, ks.clone()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,new,past", [(24, 8, [1], [516]), (3, 1, [70, 0, 1, 130], [0, 5, 63, 60]),
                                            (16, 2, [1] * 40, list(range(40))), (5, 5, [300], [1])])
def test_store_and_read(cuda_device, device_checks, kind, dtype, hq, hk, new, past):
    dev, total = cuda_device, sum(new)
    g = torch.Generator(device=dev).manual_seed(total)
    bt, cu, ctx, nb, (page, place) = batch(dev, new, past)
    qkv = torch.randn(total, hq + 2 * hk, 128, generator=g, device=dev)
    qkv = (qkv * torch.exp(3 * torch.randn(total, hq + 2 * hk, 1, generator=g, device=dev))).to(dtype)
    cos, sin = tables(dev)
    pos = torch.randint(0, 5000, (1, total), generator=g, device=dev, dtype=torch.int32)
    pos[0, ::3] = 0
    k, v, ks, vs = pools(dev, nb, hk, kind)
    q = rope_axes_store(qkv.view(total, -1), hq, cos, sin, pos, (64,), k, v, bt, 64, cu, ctx, k_scale=ks, v_scale=vs)
    # q as without codes
    k16, v16 = (torch.zeros(nb, 64, hk, 128, dtype=dtype, device=dev) for _ in "kv")
    q16 = rope_axes_store(qkv.view(total, -1), hq, cos, sin, pos, (64,), k16, v16, bt, 64, cu, ctx)
    assert torch.equal(q, q16)
    got_v, got_vs = v[page, place].double(), vs[page, :, place]
    code, scale, _ = exact_codes(qkv[:, hq + hk:], kind)
    assert torch.equal(got_v, code) and torch.equal(got_vs, scale.float())
    x = qkv[:, hq:hq + hk].double()
    still = pos[0] == 0
    code, scale, _ = exact_codes(qkv[still][:, hq:hq + hk], kind)
    assert torch.equal(k[page, place].double()[still], code) and torch.equal(ks[page, :, place][still], scale.float())
    c, s = (t.double()[pos[0].long()][:, None] for t in (cos, sin))
    rot = x * c + torch.cat([-x[..., 64:], x[..., :64]], -1) * s
    code, scale, step = exact_codes(rot, kind)
    top_code = CODES[kind][1]
    slack = 4e-5 * top_code / 127 + 0.5 * step
    z = rot * top_code / rot.abs().amax(-1, keepdim=True)
    assert ((k[page, place].double() - z).abs() <= slack).all()
    assert ((ks[page, :, place].double() - scale).abs() <= 2.0 ** -21 * scale).all()
    # slots of no new token stay as they were
    rest = torch.ones(nb, 64, dtype=torch.bool, device=dev)
    rest[page, place] = False
    assert (k.float()[rest] == 3).all() and (ks.transpose(1, 2)[rest] == 7).all()
    # read back: code * scale in fp32, rounded once
    for out in (torch.float16, torch.bfloat16):
        rk, rv = read_kv(k, v, ks, vs, bt, 64, cu, ctx, total, dtype=out)
        assert torch.equal(rk, (k[page, place].float() * ks[page, :, place][..., None]).to(out))
        assert torch.equal(rv, (v[page, place].float() * vs[page, :, place][..., None]).to(out))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_rows_of_zeros_ties_extremes_and_nan(cuda_device, kind):
    dev, rows = cuda_device, 12
    bt, cu, ctx, nb, (page, place) = batch(dev, [rows], [3])
    cos, sin = tables(dev, 2)
    pos = torch.zeros(1, rows, dtype=torch.int32, device=dev)
    for dtype in (torch.float16, torch.bfloat16):
        x = torch.randn(rows, 3, 128, device=dev).to(dtype)
        x[0] = 0
        x[1, :, :64], x[1, :, 64:] = 1.0, 0.5                # 63.5 codes: a tie, to even
        x[2] = torch.finfo(dtype).max
        x[3] = torch.finfo(dtype).tiny
        x[4, :, 5] = math.nan
        x[5, :, 127] = -math.inf
        x[6] = torch.finfo(dtype).max * torch.rand(3, 128, device=dev).to(dtype)
        x[7, :, :] = 0
        x[7, :, 9] = -3.0
        x[8] = x[8] * 1e-6
        if dtype == torch.bfloat16:
            x[9] = x[9] * 1e34
            x[10] = x[10] * 1e-30
        k, v, ks, vs = pools(dev, nb, 1, kind)
        rope_axes_store(x.view(rows, -1), 1, cos, sin, pos, (64,), k, v, bt, 64, cu, ctx, k_scale=ks, v_scale=vs)
        good = [r for r in range(rows) if r not in (4, 5)]
        for pool, scales, h in ((k, ks, 1), (v, vs, 2)):
            code, scale, _ = exact_codes(x[good, h], kind)
            assert torch.equal(pool[page, place, 0].double()[good], code)
            assert torch.equal(scales[page, 0, place][good], scale.float())
            assert torch.isnan(scales[page, 0, place][[4, 5]]).all()
        rk, rv = read_kv(k, v, ks, vs, bt, 64, cu, ctx, rows, dtype=dtype)
        assert torch.isnan(rk[[4, 5]]).all() and torch.isnan(rv[[4, 5]]).all()
        assert torch.isfinite(rk[good]).all() and (rk[0] == 0).all()


def test_missing_pages_and_rows_outside(cuda_device):
    """A slot without a page is not written and reads as zero, and device checks say so; rows of no sequence stay."""
    dev = cuda_device
    cos, sin = tables(dev, 2)
    cu = torch.tensor([1, 4], dtype=torch.int32, device=dev)
    ctx = torch.tensor([66], dtype=torch.int32, device=dev)  # slots 63, 64, 65
    bt = torch.tensor([[1, 9]], dtype=torch.int32, device=dev)
    qkv = torch.randn(6, 3 * 128, device=dev).half()
    pos = torch.zeros(1, 6, dtype=torch.int32, device=dev)
    k, v, ks, vs = pools(dev, 3, 1, "int8")
    q = torch.full((6, 1, 128), 5.0, device=dev).half()
    rope_axes_store(qkv, 1, cos, sin, pos, (64,), k, v, bt, 64, cu, ctx, q, k_scale=ks, v_scale=vs)
    assert (q[[0, 4, 5]] == 5).all() and (ks != 7).sum().item() == 1 and ks[1, 0, 63] != 7
    rk, rv = read_kv(k, v, ks, vs, bt, 64, cu, ctx, 6)
    assert (rk[2:4] == 0).all() and (rv[2:4] == 0).all() and (rk[1] != 0).any()
    from fast_infer_b200._runtime import device_checks
    with device_checks(True):
        with pytest.raises(RuntimeError, match="page pool"):
            rope_axes_store(qkv, 1, cos, sin, pos, (64,), k, v, bt, 64, cu, ctx, k_scale=ks, v_scale=vs)
        with pytest.raises(RuntimeError, match="page pool"):
            read_kv(k, v, ks, vs, bt, 64, cu, ctx, 6)


def test_strided_pools(cuda_device, device_checks):
    """Pools and scales that are views: K and V of one allocation, heads outermost."""
    dev = cuda_device
    new, past, hk = [40, 3], [30, 0], 3
    bt, cu, ctx, nb, _ = batch(dev, new, past)
    cos, sin = tables(dev, 2)
    qkv = torch.randn(43, (4 + 2 * hk) * 128, device=dev).half()
    pos = torch.zeros(1, 43, dtype=torch.int32, device=dev)
    dense = pools(dev, nb, hk, "int8")
    rope_axes_store(qkv, 4, cos, sin, pos, (64,), *dense[:2], bt, 64, cu, ctx, k_scale=dense[2], v_scale=dense[3])
    both = torch.full((hk, nb, 64, 256), 3, device=dev).to(torch.int8)
    k, v = both[..., :128].permute(1, 2, 0, 3), both[..., 128:].permute(1, 2, 0, 3)
    sc = torch.full((64, hk, nb, 2), 7.0, device=dev)
    ks, vs = sc[..., 0].permute(2, 1, 0), sc[..., 1].permute(2, 1, 0)
    rope_axes_store(qkv, 4, cos, sin, pos, (64,), k, v, bt, 64, cu, ctx, k_scale=ks, v_scale=vs)
    for a, b in zip((k, v, ks, vs), dense):
        assert torch.equal(a, b)
    for a, b in zip(read_kv(k, v, ks, vs, bt, 64, cu, ctx, 43), read_kv(*dense, bt, 64, cu, ctx, 43)):
        assert torch.equal(a, b)
