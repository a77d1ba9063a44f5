"""Numbers at the edges of what accept_drafts and sample_tokens take."""

import pytest
import torch

from fast_infer_b200.kernels.drafting import accept_drafts
from fast_infer_b200.kernels.sampling import sample_tokens

pytestmark = pytest.mark.gpu


def test_no_draft_is_accepted_after_a_row_without_a_token(cuda_device, device_checks):
    """-1 is no token: a draft of -1 (padding) does not follow a row that gave -1, in the first 32 nodes or past them."""
    dev = cuda_device
    for n, child in ((5, 1), (5, 4), (70, 1), (70, 40), (70, 69)):
        par = torch.full((n,), -1, dtype=torch.int32, device=dev)
        tok = torch.full((n,), -1, dtype=torch.int32, device=dev)
        smp = torch.full((n,), -1, dtype=torch.int32, device=dev)
        cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
        par[child] = 0
        path, counts, follow = accept_drafts(tok, smp, par, cu)
        assert (counts.tolist(), follow.tolist()) == ([1], [-1])
        assert path.tolist() == [0] + [-1] * (n - 1)
        tok[child] = smp[0] = 0  # (token 0 is one)
        path, counts, follow = accept_drafts(tok, smp, par, cu)
        assert (counts.tolist(), follow.tolist()) == ([2], [-1]) and path[:2].tolist() == [0, child]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_top_k_past_32_bits(cuda_device, dtype):
    """top_k of 64 bits keeps what it says: more than there are keeps all, and so does a negative number."""
    x = torch.zeros(4, 1000, dtype=dtype, device=cuda_device)
    u = torch.full((4,), 0.9995, device=cuda_device)
    k = torch.tensor([2 ** 32 + 1, 2 ** 31, 2 ** 63 - 1, 7], device=cuda_device)
    assert sample_tokens(x, u, top_k=k).tolist() == [999, 999, 999, 6]
    assert sample_tokens(x, u, top_k=torch.tensor([5 - 2 ** 32, -1, 0, 1], device=cuda_device)).tolist() == [999, 999, 999, 0]
    for one, want in ((2 ** 32 + 1, 999), (2 ** 64 + 3, 999), (3, 2)):
        assert sample_tokens(x, u, top_k=one).tolist() == [want] * 4
