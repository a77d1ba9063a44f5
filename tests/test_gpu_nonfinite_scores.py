"""Infinite and NaN keys, queries and lse that are seen: a score of -inf has weight 0, a NaN or +inf one makes NaN of
the rows that see it and of no other, in both forms of the attention kernel and in the weights received."""

import math

import pytest
import torch

from tests.test_gpu_attention_mass import check as check_mass
from tests.test_gpu_attention_mass import oracle_mass
from tests.test_gpu_attention_mass import run as run_mass
from tests.test_gpu_paged_chunk import PAGE, check, make, oracle, run

pytestmark = pytest.mark.gpu


def slot(batch, b, j):
    """(page, row) of token j of sequence b."""
    return int(batch[3][b, j // PAGE]), j % PAGE


def positive(batch):
    """The batch with a first dim of q, changed in place, that makes q.k = -inf in every row where k[0] = -inf."""
    batch[0][..., 0] = batch[0][..., 0].abs() + 0.5
    return batch


def hide(batch, b, keys):
    for j in keys:
        batch[1][slot(batch, b, j)][..., 0] = -math.inf


def reference(batch):
    """The definition in 64 bits, with infinities as they are: (o, lse, weight of |v|)."""
    q, k, v, table, cu, ctx = batch
    total, hq, d = q.shape
    hk = k.shape[2]
    o, absv = (torch.zeros(total, hq, d, dtype=torch.float64) for _ in range(2))
    lse = torch.full((total, hq), -math.inf, dtype=torch.float64)
    for b, n in enumerate(ctx.tolist()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        j = torch.arange(n)
        pages = table[b, j // PAGE].long()
        kb, vb = k[pages, j % PAGE].double(), v[pages, j % PAGE].double()
        see = j <= torch.arange(n - (hi - lo), n)[:, None]
        for h in range(hq):
            kh = h // (hq // hk)
            # (elementwise: a matrix product may not say what 0 * inf is)
            s = (q[lo:hi, None, h].double() * kb[None, :, kh]).sum(-1) * d ** -0.5
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True)
            e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            l = e.sum(-1, keepdim=True)
            w = e / torch.where(l == 0, 1.0, l)
            o[lo:hi, h], absv[lo:hi, h] = w @ vb[:, kh], w @ vb[:, kh].abs()
            lse[lo:hi, h] = (torch.where(top == -math.inf, 0.0, top) + torch.log(l))[:, 0]
    return o, lse, absv


def agree(got, ref, dtype=torch.float16):
    """NaN exactly where the definition has NaN; elsewhere the attention tests' tolerance."""
    out, lse = got
    nan = torch.isnan(ref[1])
    assert torch.equal(torch.isnan(lse.cpu()), nan)
    assert torch.equal(torch.isnan(out.cpu()).all(-1), nan) and torch.equal(torch.isnan(out.cpu()).any(-1), nan)
    if not nan.all():
        rows = ~nan.any(-1)
        check(out.cpu()[rows], lse.cpu()[rows], tuple(x[rows] for x in ref), dtype)


# Which keys of the last sequence score -inf: the newest alone in its tile, a whole first tile, all but the newest, all,
# a few anywhere, the second warpgroup's first tile.
HIDDEN = {"newest_alone": (129, [128]), "first_tile": (300, range(128)), "all_but_newest": (260, range(259)),
          "all": (140, range(140)), "some": (400, [0, 1, 16, 130, 399]), "second_tile": (384, range(128, 256))}


@pytest.mark.parametrize("hq,hk,new", [(2, 1, 1), (6, 2, 5), (6, 2, 90), (8, 8, 33)])
@pytest.mark.parametrize("name", list(HIDDEN))
def test_keys_that_score_minus_infinity_have_weight_zero(cuda_device, device_checks, name, hq, hk, new):
    ctx, keys = HIDDEN[name]
    batch = positive(make([(new, 200), (new, ctx)], hq, hk, torch.float16))
    hide(batch, 1, keys)
    agree(run(batch, cuda_device), reference(batch))


@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("name", list(HIDDEN))
def test_keys_that_score_minus_infinity_in_a_whole_unit(cuda_device, device_checks, name, new):
    """So many sequences that a CTA has all key tiles of a unit: its two warpgroups merge their rows."""
    ctx, keys = HIDDEN[name]
    batch = positive(make([(new, ctx)] * 300, 2, 1, torch.float16))
    for b in range(0, 300, 3):
        hide(batch, b, keys)
    agree(run(batch, cuda_device), reference(batch))


def test_key_that_scores_plus_infinity_shows(cuda_device, device_checks):
    for hq, hk, new, ctx, j in ((2, 1, 1, 129, 128), (2, 1, 1, 300, 3), (6, 2, 90, 300, 250), (6, 2, 90, 300, 256)):
        batch = positive(make([(new, ctx)], hq, hk, torch.float16))
        batch[1][slot(batch, 0, j)][..., 0] = math.inf
        agree(run(batch, cuda_device), reference(batch))


@pytest.mark.parametrize("hq,hk,new,ctx", [(2, 1, 1, 700), (6, 2, 4, 300), (6, 2, 90, 300), (6, 2, 300, 900)])
def test_nan_query_shows_in_its_rows_alone(cuda_device, device_checks, hq, hk, new, ctx):
    batch = make([(new, ctx), (new, 70)], hq, hk, torch.float16, garbage=0.0)
    batch[0][new - 1, 1, 5] = math.nan
    agree(run(batch, cuda_device), reference(batch))


@pytest.mark.parametrize("hq,hk,new,ctx,j", [
    (2, 1, 1, 1, 0), (6, 2, 3, 3, 0), (6, 2, 90, 90, 0),  # the only key that the first token sees
    (2, 1, 1, 129, 128), (2, 1, 2, 130, 128), (6, 2, 60, 257, 256),  # alone in the last tile of a cut unit
    (2, 1, 1, 385, 384), (2, 1, 1, 385, 130), (2, 1, 1, 385, 0)])
def test_nan_key_shows_in_every_row_that_sees_it(cuda_device, device_checks, hq, hk, new, ctx, j):
    batch = make([(new, ctx)], hq, hk, torch.float16, garbage=0.0)
    batch[1][slot(batch, 0, j)] = math.nan
    agree(run(batch, cuda_device), reference(batch))


@pytest.mark.parametrize("j", list(range(144, 160)))
def test_nan_key_shows_at_every_column(cuda_device, device_checks, j):
    """Wide units, whose columns take two forms of exp2 in turn."""
    batch = make([(90, 300)], 6, 2, torch.float16, garbage=0.0)
    batch[1][slot(batch, 0, j)][1, 7] = math.nan  # one KV head of two
    agree(run(batch, cuda_device), reference(batch))


def mass_with_nan(batch, lse, dev, nan_keys=(), nan_rows=()):
    """Weights of a batch whose one sequence has a NaN key or NaN rows: NaN there and right elsewhere."""
    q, k, v, table, cu, ctx = batch
    got = run_mass(batch, dev, lse).cpu()
    hq, hk = q.shape[1], k.shape[2]
    new, n = q.shape[0], int(ctx[0])
    nan = torch.zeros(got.shape, dtype=torch.bool)
    for j in nan_keys:
        nan[0, :, j] = True
    for i, h in nan_rows:
        nan[0, h // (hq // hk), :n - new + i + 1] = True
    assert torch.equal(torch.isnan(got), nan)
    clean = (torch.nan_to_num(q), torch.nan_to_num(k), v, table, cu, ctx)
    ref = oracle_mass(clean, torch.nan_to_num(lse))
    check_mass(torch.where(nan, 0.0, got), torch.where(nan, 0.0, ref))


@pytest.mark.parametrize("hq,hk,new", [(1, 1, 1), (2, 1, 1), (2, 2, 2), (6, 2, 5), (6, 2, 90), (8, 1, 40)])
def test_nan_in_mass_shows(cuda_device, device_checks, hq, hk, new):
    """A NaN key makes NaN of its own weight, a NaN query row or lse of the keys that the row sees."""
    ctx = 300
    base = make([(new, ctx)], hq, hk, torch.float16, garbage=0.0)
    lse = oracle(base)[1].float()
    for j in (0, ctx - new, 131):
        if j > ctx - new:
            continue
        batch = tuple(t.clone() for t in base)
        batch[1][slot(batch, 0, j)] = math.nan
        mass_with_nan(batch, lse, cuda_device, nan_keys=[j])
    for i, h in ((0, 0), (new - 1, hq - 1), (new // 2, hq // 2)):
        bad = lse.clone()
        bad[i, h] = math.nan
        mass_with_nan(base, bad, cuda_device, nan_rows=[(i, h)])
        batch = tuple(t.clone() for t in base)
        batch[0][i, h, 77] = math.nan
        mass_with_nan(batch, lse, cuda_device, nan_rows=[(i, h)])


@pytest.mark.parametrize("hq,hk,new", [(1, 1, 1), (6, 2, 5), (6, 2, 90), (7, 1, 90), (8, 8, 200)])
def test_mass_of_keys_that_score_minus_infinity_is_zero(cuda_device, device_checks, hq, hk, new):
    """Groups whose tiles do not fill 128 rows among them: the columns left over hold products with 0."""
    batch = positive(make([(new, 700)], hq, hk, torch.float16, garbage=0.0))
    lse = oracle(batch)[1].float()
    ref = oracle_mass(batch, lse)
    keys = [0, 3, 100, 255, 400]
    hide(batch, 0, keys)
    ref[0, :, keys] = 0.0
    check_mass(run_mass(batch, cuda_device, lse), ref)


@pytest.mark.parametrize("hq", [1, 2, 16, 17])
def test_mass_past_fp32_is_infinite(cuda_device, device_checks, hq):
    """An lse far below the scores (of a call with a narrower mask, say): weights past fp32 are +inf, not wrapped; those
    below it hold."""
    batch = make([(1, 200)], hq, 1, torch.float16, garbage=0.0)
    lse = oracle(batch)[1].float()
    got = run_mass(batch, cuda_device, lse - 60.0).cpu()
    check_mass(got, oracle_mass(batch, lse - 60.0), 8.0)  # arguments of up to 2^7 in log2 units
    for down in (200.0, 1000.0, 1e30, math.inf):
        row = (lse - down) if down < math.inf else torch.full_like(lse, -3e38)
        got = run_mass(batch, cuda_device, row).cpu()
        assert (got[0, 0, :200] == math.inf).all() and not got[0, 0, 200:].any()
