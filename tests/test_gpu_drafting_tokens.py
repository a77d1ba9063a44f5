"""Numbers at the edges of what accept_drafts and sample_tokens take."""

import pytest
import torch

from fast_infer_b200.kernels.drafting import accept_drafts

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
