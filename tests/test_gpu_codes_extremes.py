"""paged_tree_attention over 8-bit codes where V's scales are far apart: rows of zeros and subnormal rows that hold most of a
softmax's weight, and rows past fp16's range. Finite caches give finite outputs, close to the definition in 64 bits,
whatever the number of rows that share a tile."""

import math

import pytest
import torch

from fast_infer_b200.kernels.attention import paged_tree_attention
from tests.test_gpu_paged_tree import check, make

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
