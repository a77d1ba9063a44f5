"""Eviction with a mass that is shorter than a sequence: cut there, as documented, and reported by device checks."""

import pytest
import torch

from tests.test_gpu_evict import make, oracle, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,rows", [([300, 90], 1), ([300, 90] * 20, 10)])
def test_short_mass_is_cut_and_reported(cuda_device, lens, rows):
    """Few rows, and many (selection and move in one kernel)."""
    from fast_infer_b200._runtime import device_checks as checks
    from fast_infer_b200.kernels.eviction import evict_tokens
    k, v, table, n, mass = make(lens, 2, rows, seed=5, cap=200)
    cut = n.clamp(max=200)
    ref = oracle((k, v, table, cut, mass), 100, 10, 4, (k, v, table))
    kd, vd, td, nd, md = (t.to(cuda_device) for t in (k, v, table, n, mass))
    with checks(True), pytest.raises(RuntimeError, match="context length"):
        evict_tokens(kd.clone(), vd.clone(), td, nd, md, 100, recent=10, sinks=4)
    with checks(False):
        kept, mass_out = evict_tokens(kd, vd, td, nd, md, 100, recent=10, sinks=4)
    assert same(kept, ref[0]) and torch.equal(mass_out.cpu(), ref[1]) and same(kd, ref[2]) and same(vd, ref[3])
