"""paged_tree_attention with many query heads a KV head: groups past 8 leave few tokens to a unit or a row tile, groups past
32 none to a unit of few rows."""

import pytest
import torch

from tests.test_gpu_paged_tree import check, make

pytestmark = pytest.mark.gpu
SEQS = [[(1, 300), (1, 70), (1, 1000)], [(3, 200), (5, 700), (4, 4), (0, 10)], [(45, 900), (1, 300), (20, 20)],
        [(1, 2500), (130, 400)]]


@pytest.mark.parametrize("kind", ["16bit", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(5, 1), (12, 1), (16, 1), (34, 2), (40, 2), (32, 1), (33, 1), (64, 1)])
@pytest.mark.parametrize("seqs", SEQS)
def test_groups(cuda_device, device_checks, seqs, heads, dtype, kind):
    for softcap, window, spread in ((0.0, 0, 5), (20.0, 60, 3), (0.0, 0, 0)):
        st = make(cuda_device, seqs, *heads, dtype, kind, seed=heads[0], spread=spread, window=window)
        check(st, kind, dtype, softcap, window)
