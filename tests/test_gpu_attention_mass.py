"""Attention weight per cached token against its definition in 64 bits: lengths, groups, score
forms and masks as for the attention itself, sums over several calls, keys cut between CTAs."""

import math

import pytest
import torch

from oracle.chunk_oracle import chunk, mass
from tests.test_gpu_paged_chunk import FORMS, PAGE, SEQS, make, oracle

pytestmark = pytest.mark.gpu
D = 128


def run(batch, dev, lse, mass=None, **form):
    from fast_infer_b200.kernels.attention import attention_mass
    q, k, _, table, cu, ctx = (t.to(dev) for t in batch)
    form = {n: (x.to(dev) if isinstance(x, torch.Tensor) else x) for n, x in form.items()}
    return attention_mass(q, k, table, PAGE, cu, ctx, lse.to(dev), mass=mass, **form)


def oracle_mass(batch, lse, alibi_slopes=None, prefix_lens=None, sm_scale=None, **form):
    q, k, _, table, cu, ctx = batch
    return mass(q, k, table, cu, ctx, lse, slopes=alibi_slopes, prefix=prefix_lens,
                scale=D ** -0.5 if sm_scale is None else sm_scale, **form)


def check(got, ref, amp=1.0):
    """Per value: exp2 is off by at most 2.2e-7 relative (2 ulp in the unit's approximation), its
    argument by the fp32 rounding of values of up to 2^4 * amp in log2 units and of the products'
    sums (2^-18 * amp together, times ln 2 in the result); the fp32 sums by 2^-24 a step over
    at most 2^7 steps. Together below 2^-15 * amp relative; where nothing sees, exactly 0."""
    got = got.double().cpu()
    assert (got[ref == 0] == 0).all()
    tol = ref * 2.0 ** -15 * amp + 1e-30
    assert ((got - ref).abs() <= tol).all(), float(((got - ref).abs() / ref.clamp(min=1e-30)).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", list(SEQS))
def test_lengths(cuda_device, device_checks, name, dtype):
    batch = make(SEQS[name], 6, 2, dtype)
    lse = oracle(batch)[1].float()
    check(run(batch, cuda_device, lse), oracle_mass(batch, lse))


@pytest.mark.parametrize("hq,hk", [(1, 1), (24, 8), (8, 1), (7, 1), (64, 1), (33, 1)])
def test_groups(cuda_device, device_checks, hq, hk):
    batch = make([(37, 150), (1, 260), (3, 3), (150, 640)], hq, hk, torch.float16)
    lse = oracle(batch)[1].float()
    check(run(batch, cuda_device, lse), oracle_mass(batch, lse))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", list(FORMS))
def test_forms(cuda_device, device_checks, name, dtype):
    batch = make([(1, 300), (130, 300), (7, 500), (1, 1), (90, 450), (2, 66)], 6, 2, dtype)
    lse = oracle(batch, **FORMS[name])[1].float()
    check(run(batch, cuda_device, lse, **FORMS[name]), oracle_mass(batch, lse, **FORMS[name]),
          4.0 if name == "scale" else 1.0)


def test_saturated_cap(cuda_device, device_checks):
    batch = make([(20, 200), (1, 77)], 4, 2, torch.float16, amp=30.0)
    lse = oracle(batch, softcap=2.0)[1].float()
    check(run(batch, cuda_device, lse, softcap=2.0), oracle_mass(batch, lse, softcap=2.0))


def test_rows_sum_to_one(cuda_device, device_checks):
    """With the lse of the attention call itself, every row's weights add up to one."""
    from fast_infer_b200.kernels.attention import paged_chunk_attention
    batch = make([(40, 333), (1, 700), (90, 200)], 6, 2, torch.float16)
    q, k, v, table, cu, ctx = (t.to(cuda_device) for t in batch)
    _, lse = paged_chunk_attention(q, k, v, table, PAGE, cu, ctx, return_lse=True)
    got = run(batch, cuda_device, lse).double().sum(-1).cpu()
    rows = torch.tensor([40.0, 1.0, 90.0])[:, None] * 3
    assert ((got - rows).abs() <= rows * 2e-4).all()  # exp2 in the attention: 7.5e-5


def test_adds_to_what_was_there(cuda_device, device_checks):
    """Two calls into one buffer give their sum; what no call's tokens see keeps its value, also
    past the context and in a sequence without new tokens."""
    first = make([(40, 333), (1, 500), (0, 70)], 6, 2, torch.float16)
    lse = oracle(first)[1].float()
    one = run(first, cuda_device, lse)
    start = torch.full((3, 2, 700), 0.5, device=cuda_device)
    got = run(first, cuda_device, lse, mass=start)
    assert got.data_ptr() == start.data_ptr()
    got = run(first, cuda_device, lse, mass=got)
    n = one.shape[2]
    want = 0.5 + one + one
    assert ((got[..., :n] - want).abs() <= 3 * 2.0 ** -24 * want).all()
    assert (got[..., n:] == 0.5).all() and (got[2] == 0.5).all()


def test_last_tokens_alone(cuda_device, device_checks):
    """The last 16 tokens of longer chunks: rows taken from the chunk's own q and lse."""
    batch = make([(50, 300), (20, 100)], 6, 2, torch.float16)
    q, k, v, table, cu, ctx = batch
    lse = oracle(batch)[1].float()
    rows = torch.cat([torch.arange(34, 50), torch.arange(54, 70)])
    part = (q[rows].contiguous(), k, v, table, torch.tensor([0, 16, 32]).int(), ctx)
    check(run(part, cuda_device, lse[rows]), oracle_mass(part, lse[rows]))


@pytest.mark.parametrize("garbage", [math.inf, -math.inf, 60000.0])
def test_unused_slots_and_rows_may_hold_anything(cuda_device, device_checks, garbage):
    batch = make(SEQS["mixed"] + [(1, 129)], 6, 2, torch.float16, garbage=garbage)
    lse = oracle(batch)[1].float()
    ref = oracle_mass(batch, lse)
    batch = (torch.cat([batch[0], torch.full_like(batch[0][:50], math.nan)]),) + batch[1:]
    lse = torch.cat([lse, torch.full_like(lse[:50], math.nan)])
    check(run(batch, cuda_device, lse), ref)


def test_invalid_pages_get_nothing(cuda_device):
    from fast_infer_b200._runtime import device_checks as checks
    q, k, v, table, cu, ctx = make([(3, 300), (40, 500)], 6, 2, torch.float16)
    table[0, 1], table[1, 3], table[1, 6] = -1, k.shape[0], -7
    batch = (q, k, v, table, cu, ctx)
    lse = oracle(batch)[1].float()
    check(run(batch, cuda_device, lse), oracle_mass(batch, lse))
    with checks(True), pytest.raises(RuntimeError, match="page pool"):
        run(batch, cuda_device, lse)


def test_short_capacity_is_reported(cuda_device):
    from fast_infer_b200._runtime import device_checks as checks
    batch = make([(3, 300), (40, 90)], 6, 2, torch.float16)
    lse = oracle(batch)[1].float()
    start = torch.zeros(2, 2, 130, device=cuda_device)
    with checks(True), pytest.raises(RuntimeError, match="context length"):
        run(batch, cuda_device, lse, mass=start)
    check(start, oracle_mass(batch, lse)[..., :130])


def test_same_bits_and_graph(cuda_device):
    from fast_infer_b200.kernels.attention import attention_mass
    batch = make([(300, 640), (1, 700), (90, 200)], 6, 2, torch.float16)
    lse = oracle(batch)[1].float()
    want = run(batch, cuda_device, lse)
    assert torch.equal(run(batch, cuda_device, lse), want)
    q, k, _, table, cu, ctx = (t.to(cuda_device) for t in batch)
    lse = lse.to(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention_mass(q, k, table, PAGE, cu, ctx, lse)
    for _ in range(2):
        got.fill_(-1.0)
        graph.replay()
        assert torch.equal(got, want)


def test_many_sequences(cuda_device, device_checks):
    g = torch.Generator().manual_seed(5)
    seqs = [(int(n), int(n) + int(c)) for n, c in zip(torch.randint(0, 3, (2048,), generator=g),
                                                       torch.randint(0, 40, (2048,), generator=g))]
    batch = make(seqs, 2, 1, torch.float16)
    lse = oracle(batch)[1].float()
    check(run(batch, cuda_device, lse), oracle_mass(batch, lse))


@pytest.mark.parametrize("softcap", [1e-3, 1e6])
def test_caps_far_from_the_scores(cuda_device, device_checks, softcap):
    batch = make([(20, 200), (1, 77), (100, 130)], 4, 2, torch.float16)
    lse = oracle(batch, softcap=softcap)[1].float()
    check(run(batch, cuda_device, lse, softcap=softcap), oracle_mass(batch, lse, softcap=softcap))
