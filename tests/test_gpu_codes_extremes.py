"""paged_tree_attention over 8-bit codes where scales are far apart or NaN: rows of zeros and subnormal rows that hold most of a
softmax's weight, and rows past fp16's range. Finite caches give finite outputs, close to the definition in 64 bits,
whatever the number of rows that share a tile."""

import math

import pytest
import torch

from fast_infer_b200.kernels.attention import paged_tree_attention
from tests.test_gpu_paged_tree import check, definition, make, visible

pytestmark = pytest.mark.gpu
KINDS = ["int8", "e4m3"]
# 3, 9, 24 and 48 rows of a KV head's group of three, and two row tiles; several sequences of each
SHAPES = [[(1, 300), (1, 700)], [(3, 500), (2, 90)], [(8, 513), (6, 400)], [(16, 640)], [(60, 800)], [(1, 900), (70, 300)]]


def aligned(dev, seqs, dtype, kind, seed, spread=4):
    """Scores that the first value of K's scale sets: q of all ones nearly, K random but for `peak`."""
    st = make(dev, seqs, 6, 2, dtype, kind, seed=seed, spread=spread)
    g = torch.Generator(device=dev).manual_seed(seed)
    st["q"] = (3.0 + 0.1 * torch.randn(st["q"].shape, generator=g, device=dev)).to(dtype)
    return st


def place(st, b, slot):
    return int(st["table"][b, slot // 64]), slot % 64


def peak(st, kind, b, slot, score):
    """Key `slot` of sequence b, all heads: all its values alike, such that q of threes scores about `score`."""
    page, at = place(st, b, slot)
    top = {"int8": 127, "e4m3": 448}[kind]
    st["k"][page, at] = torch.full_like(st["k"][page, at].float(), top).to(st["k"].dtype)
    st["ks"][page, :, at] = score * math.sqrt(128) / (3 * 128 * top)
    return page, at


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seqs", SHAPES)
def test_a_row_of_zeros_takes_all_weight(cuda_device, device_checks, seqs, dtype, kind):
    """A key 100 to 200 nats above the others whose V row is zero, or subnormal in fp32 terms: o is near 0, lse the key's."""
    for score, scale, softcap in ((110.0, 0.0, 0.0), (200.0, 0.0, 0.0), (140.0, 1e-41, 0.0), (95.0, 0.0, 100.0)):
        st = aligned(cuda_device, seqs, dtype, kind, seed=21)
        for x in "k":  # (other scores within a few nats)
            st[x + "s"] *= 0.1
        for b, (n, c) in enumerate(seqs):
            page, at = peak(st, kind, b, (c - n) // 2, score)
            st["vs"][page, :, at] = scale
        o, _ = check(st, kind, dtype, softcap)
        assert torch.isfinite(o).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seqs", SHAPES)
def test_subnormal_rows_come_first(cuda_device, device_checks, seqs, dtype, kind):
    """V rows near 1e-38 in the first pages, or everywhere, ordinary ones behind them."""
    for pages in (1, 2, 3, 10 ** 6):
        st = make(cuda_device, seqs, 6, 2, dtype, kind, seed=22, spread=4)
        for b in range(len(seqs)):
            for page in st["table"][b, :pages].tolist():
                if page >= 0:
                    st["vs"][page] *= 1e-38
        o, _ = check(st, kind, dtype)
        assert torch.isfinite(o).all()


def bound(st, dtype, softcap, window):
    """Exact o, lse, and how far o may be off. Weights times V's scales are rounded to 16 bits relative to a running maximum
    of theirs, which lies at 2^5 or above: a key adds half a step of its own or 2^-25 / 2^5 of the row's greatest p max|v|."""
    exact, absv, _, lse, err = definition(st, softcap, window)
    eps = torch.finfo(dtype).eps / 2
    least = torch.zeros_like(lse)
    row = 0
    for b, ((n, c), see) in enumerate(zip(st["seqs"], visible(st, window))):
        pages = st["table"][b, :-(-c // 64)].long()
        if n == 0 or c == 0:
            row += n
            continue
        for h in range(st["q"].shape[1]):
            kh = h // (st["q"].shape[1] // st["k"].shape[2])
            k = (st["k"][pages][:, :, kh].double() * st["ks"][pages, kh].double()[..., None]).reshape(-1, 128)[:c]
            v = (st["v"][pages][:, :, kh].double() * st["vs"][pages, kh].double()[..., None]).reshape(-1, 128)[:c]
            s = st["q"][row:row + n, h].double() @ k.t() / math.sqrt(128)
            s = softcap * torch.tanh(s / softcap) if softcap else s
            p = torch.exp(s.masked_fill(~see.to(s.device), -math.inf) - lse[row:row + n, h, None])
            least[row:row + n, h] = c * 2.0 ** -30 * (p * v.abs().amax(-1)).amax(-1)
        row += n
    tol = (2 * eps * 1.01 + 2 * err[..., None]) * absv + eps * exact.abs() + least[..., None]
    return exact, lse, tol + (2.0 ** -25 if dtype == torch.float16 else 1e-30), err


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seqs", SHAPES + [[(1, 4)], [(5, 5)], [(2, 9000)]])
def test_scales_six_orders_apart(cuda_device, device_checks, seqs, dtype, kind):
    """V rows up to 10^6 apart in size: where the greatest row's values are 0, the small ones are what counts."""
    for seed, softcap, window in ((1, 0.0, 0), (2, 30.0, 40)):
        st = make(cuda_device, seqs, 6, 2, dtype, kind, seed=seed, spread=4, window=window)
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        st["vs"] *= 10.0 ** (6 * torch.rand(st["vs"].shape, generator=g, device=cuda_device) - 6)
        st["v"].view(torch.int8)[torch.rand(st["v"].shape, generator=g, device=cuda_device) < 0.2] = 0
        exact, exact_lse, tol, err = bound(st, dtype, softcap, window)
        o, lse = paged_tree_attention(st["q"], st["k"], st["v"], st["table"], 64, st["cu"], st["ctx"], tree_mask=st["mask"],
                                      depths=st["depths"], k_scale=st["ks"], v_scale=st["vs"], softcap=softcap, window=window,
                                      return_lse=True)
        assert ((lse.double() - exact_lse).abs() <= err + 2.0 ** -22 * exact_lse.abs()).all()
        far = (o.double() - exact).abs()
        assert (far <= tol).all(), (far / tol).max()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seqs", SHAPES)
def test_rows_past_the_range_of_fp16(cuda_device, device_checks, seqs, dtype, kind):
    """V rows of 1e10 at keys of little weight count for what they are; those of 1e30 at a new token do not show in rows that do
    not see it."""
    top = {"int8": 127.0, "e4m3": 448.0}[kind]
    for softcap, score, size in ((0.0, -20.0, 1e10), (30.0, -27.0, 1e11), (0.0, -9.0, 1e6)):
        st = aligned(cuda_device, seqs, dtype, kind, seed=23)
        st["ks"] *= 0.1
        for b, (n, c) in enumerate(seqs):
            for slot in {c - n - 1, (c - n) // 3}:
                page, at = peak(st, kind, b, slot, score)
                st["vs"][page, :, at] = size / top
            if n > 2:  # (a sibling's key: no other branch sees it)
                page, at = place(st, b, c - n + 2)
                st["vs"][page, :, at] = 1e30
        exact, exact_lse, tol, err = bound(st, dtype, softcap, 0)
        o, lse = paged_tree_attention(st["q"], st["k"], st["v"], st["table"], 64, st["cu"], st["ctx"], tree_mask=st["mask"],
                                      k_scale=st["ks"], v_scale=st["vs"], softcap=softcap, return_lse=True)
        assert ((lse.double() - exact_lse).abs() <= err + 2.0 ** -22 * exact_lse.abs()).all()
        ok = exact.abs().amax(-1) < 3e4  # (rows that see the 1e30 are past fp16)
        assert ok.any(-1).sum() >= len(seqs)
        far = (o.double() - exact).abs()
        assert (far <= tol)[ok].all(), (far / tol)[ok].max()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seqs", [[(16, 640)], [(60, 800)], [(2, 300), (70, 5000)]])
def test_nan_scores_show_in_the_rows_that_see_them(cuda_device, seqs, dtype, kind):
    """A NaN scale of a new token's K: NaN in o and lse of the rows that see that key, finite elsewhere."""
    st = make(cuda_device, seqs, 6, 2, dtype, kind, seed=24, spread=4)
    row = 0
    sees = torch.zeros(st["q"].shape[0], dtype=torch.bool)
    for b, ((n, c), see) in enumerate(zip(seqs, visible(st, 0))):
        page, at = place(st, b, c - n + n // 2)
        st["ks"][page, 1, at] = math.nan
        sees[row:row + n] = see[:, c - n + n // 2]
        row += n
    o, lse = paged_tree_attention(st["q"], st["k"], st["v"], st["table"], 64, st["cu"], st["ctx"], tree_mask=st["mask"],
                                  k_scale=st["ks"], v_scale=st["vs"], return_lse=True)
    sees = sees.to(cuda_device)
    assert sees.any() and not sees.all()
    assert torch.isnan(o[sees][:, 3:]).all() and torch.isnan(lse[sees][:, 3:]).all()
    assert torch.isfinite(o[~sees]).all() and torch.isfinite(lse[~sees]).all() and torch.isfinite(o[:, :3]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(64, 1), (33, 1), (24, 8)])
def test_lse_of_few_small_scores(cuda_device, device_checks, heads, dtype, kind):
    """One or two keys with scores near 0: lse is as exact as fp32 sums, whatever V's scales are."""
    st = make(cuda_device, [(1, 1), (2, 2), (1, 2)] * 8, *heads, dtype, kind, seed=25, spread=3)
    st["ks"] *= 1e-3
    check(st, kind, dtype)
