"""Attention of new tokens over the paged cache against its definition in 64 bits: lengths from
none to several tiles, groups of query heads, every score form and mask, pages in any order,
garbage in unused slots, strides, streams and captured graphs."""

import math

import pytest
import torch

from oracle.chunk_oracle import chunk

pytestmark = pytest.mark.gpu
PAGE, D = 64, 128


def make(seqs, hq, hk, dtype, seed=0, spare=3, garbage=math.nan, amp=1.0):
    """CPU tensors of a batch: seqs = [(new tokens, cached tokens with them)]. Slots and pages that
    no token owns hold `garbage`."""
    g = torch.Generator().manual_seed(seed)
    pages = [max(0, (c + PAGE - 1) // PAGE) for _, c in seqs]
    nb = sum(pages) + spare
    order = torch.randperm(nb, generator=g).int()
    table = torch.full((len(seqs), max(pages + [0]) + 2), -1, dtype=torch.int32)
    k = torch.full((nb, PAGE, hk, D), garbage, dtype=dtype)
    v = torch.full((nb, PAGE, hk, D), garbage, dtype=dtype)
    at = 0
    for b, (_, c) in enumerate(seqs):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
        for i in range(pages[b]):
            n = min(PAGE, c - i * PAGE)
            page = int(table[b, i])
            k[page, :n] = torch.randn(n, hk, D, generator=g).to(dtype)
            v[page, :n] = torch.randn(n, hk, D, generator=g).to(dtype)
    new = [n for n, _ in seqs]
    q = (torch.randn(sum(new), hq, D, generator=g) * amp).to(dtype)
    cu = torch.tensor([0] + new).cumsum(0).int()
    return q, k, v, table, cu, torch.tensor([c for _, c in seqs]).int()


def check(out, lse, ref, dtype, amp=1.0):
    """The tolerance, per value: P and o are rounded to `dtype` once each (half a step, u, relative:
    u * (sum p |v| + |o|)); exp2 is off by at most 7.5e-5 relative, in numerator and denominator; a
    score (fp32 products and sums over 128 dims, |q||k| sums of at most ~2^8 * amp in scaled units
    of 0.088) by at most 2^-14 * amp absolute with the cap's polynomial; P below 2^-14 loses at
    most 2^-25 a key in fp16."""
    o, l, absv = ref
    u = torch.finfo(dtype).eps / 2
    rel = 2 * 7.5e-5 + 2 * 2.0 ** -14 * amp
    tol = u * (absv + o.abs()) + rel * absv + 2.0 ** -25 * 16 * o.shape[0] + 1e-7
    diff = (out.double().cpu() - o).abs()
    assert torch.isfinite(out.double()).all()
    assert (diff <= tol).all(), f"o: {float((diff - tol).max()):.3e} past the tolerance"
    empty = torch.isinf(l)
    got = lse.double().cpu()
    assert torch.equal(torch.isinf(got), empty) and (got[empty] < 0).all()
    assert not out.cpu()[empty].any()
    ltol = 7.5e-5 + 2.0 ** -14 * amp + l[~empty].abs() * 2.0 ** -22
    assert ((got - l)[~empty].abs() <= ltol).all(), float((got - l)[~empty].abs().max())


def run(batch, dev, **form):
    from fast_infer_b200.kernels.attention import paged_chunk_attention
    q, k, v, table, cu, ctx = (t.to(dev) for t in batch)
    form = {n: (x.to(dev) if isinstance(x, torch.Tensor) else x) for n, x in form.items()}
    return paged_chunk_attention(q, k, v, table, PAGE, cu, ctx, return_lse=True, **form)


def oracle(batch, alibi_slopes=None, prefix_lens=None, sm_scale=None, **form):
    return chunk(*batch, slopes=alibi_slopes, prefix=prefix_lens,
                 scale=D ** -0.5 if sm_scale is None else sm_scale, **form)


SEQS = {
    "one": [(1, 1)],
    "one_token": [(1, 517)],
    "whole_prompt": [(200, 200)],
    "page_edges": [(1, 64), (1, 65), (64, 128), (65, 129), (3, 63)],
    "tile_edges": [(42, 128), (43, 129), (84, 300), (85, 257)],
    "none_among": [(0, 0), (5, 70), (0, 33), (1, 1), (0, 128)],
    "long_chunk": [(300, 700)],
    "decode_batch": [(1, c) for c in (1, 63, 64, 65, 400, 129, 250, 7, 191, 320)],
    "mixed": [(1, 300), (130, 131), (7, 500), (1, 1), (90, 90), (2, 66)],
    "few_tokens_but_one": [(1, 100)] * 9 + [(60, 300), (0, 5)],
    "many_tokens_in_one": [(1, 70)] * 70 + [(600, 650), (0, 9), (15, 40)],
    "many_tokens_in_few_rows_each": [(9, 30 + i) for i in range(80)],
    "cached_missing": [(5, 3), (4, 0), (150, 100)],  # fewer cached tokens than new ones
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", list(SEQS))
def test_lengths(cuda_device, device_checks, name, dtype):
    batch = make(SEQS[name], 6, 2, dtype)
    check(*run(batch, cuda_device), oracle(batch), dtype)


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (24, 8), (8, 1), (20, 4), (7, 1), (64, 1), (33, 1)])
def test_groups(cuda_device, device_checks, hq, hk):
    batch = make([(37, 150), (1, 260), (3, 3)], hq, hk, torch.float16)
    check(*run(batch, cuda_device), oracle(batch), torch.float16)


SLOPES = torch.tensor([0.5, 0.25, 0.0, 0.0625, 1.0, 0.01])
FORMS = {
    "cap": dict(softcap=5.0),
    "cap_small_scores": dict(softcap=50.0),
    "alibi": dict(alibi_slopes=SLOPES),
    "cap_alibi": dict(softcap=20.0, alibi_slopes=SLOPES),
    "window": dict(window=100),
    "window_one": dict(window=1),
    "prefix": dict(prefix_lens=torch.tensor([0, 200, 1, 5000, 17, 64], dtype=torch.int32)),
    "window_prefix": dict(window=70, prefix_lens=torch.tensor([3, 130, 0, 9, 400, 65], dtype=torch.int32)),
    "all": dict(softcap=10.0, alibi_slopes=SLOPES, window=33,
                prefix_lens=torch.tensor([3, 130, 0, 9, 400, 65], dtype=torch.int32)),
    "scale": dict(sm_scale=0.3),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", list(FORMS))
def test_forms(cuda_device, device_checks, name, dtype):
    batch = make([(1, 300), (130, 300), (7, 500), (1, 1), (90, 450), (2, 66)], 6, 2, dtype)
    amp = 0.3 / D ** -0.5 if name == "scale" else 1.0
    check(*run(batch, cuda_device, **FORMS[name]), oracle(batch, **FORMS[name]), dtype, amp)


def test_saturated_cap(cuda_device, device_checks):
    """Scores far past the cap: tanh at its ends, equal weights."""
    batch = make([(20, 200), (1, 77)], 4, 2, torch.float16, amp=30.0)
    check(*run(batch, cuda_device, softcap=2.0), oracle(batch, softcap=2.0), torch.float16, 30.0)


def test_large_scores(cuda_device, device_checks):
    """Scores of a few hundred: the running maximum moves, weights underflow."""
    batch = make([(64, 640), (1, 500)], 4, 2, torch.float16, amp=25.0)
    check(*run(batch, cuda_device), oracle(batch), torch.float16, 25.0)


@pytest.mark.parametrize("garbage", [math.inf, -math.inf, 60000.0])
def test_unused_slots_may_hold_anything(cuda_device, device_checks, garbage):
    batch = make(SEQS["mixed"] + [(1, 129)], 6, 2, torch.float16, garbage=garbage)
    check(*run(batch, cuda_device), oracle(batch), torch.float16)


def test_invalid_pages_are_skipped_and_reported(cuda_device):
    from fast_infer_b200._runtime import device_checks as checks
    q, k, v, table, cu, ctx = make([(3, 300), (40, 500)], 6, 2, torch.float16)
    nb = k.shape[0]
    table[0, 1], table[1, 3], table[1, 6] = -1, nb, -7
    batch = (q, k, v, table, cu, ctx)
    check(*run(batch, cuda_device), oracle(batch), torch.float16)
    with checks(True), pytest.raises(RuntimeError, match="page pool"):
        run(batch, cuda_device)


def test_lengths_beyond_the_table_are_cut_and_reported(cuda_device):
    from fast_infer_b200._runtime import device_checks as checks
    q, k, v, table, cu, ctx = make([(2, 128), (3, 64)], 6, 2, torch.float16)
    table = table[:, :2].contiguous()
    long = ctx.clone()
    long[0] = 400  # positions 398, 399: both see every key that the table holds
    with checks(True), pytest.raises(RuntimeError, match="context length"):
        run((q, k, v, table, cu, long), cuda_device)
    with checks(True), pytest.raises(RuntimeError, match="context length"):
        run((q, k, v, table, torch.tensor([0, 4, 2]).int(), ctx), cuda_device)
    out, lse = run((q, k, v, table, cu, long), cuda_device)
    ref = oracle((q, k, v, table, cu, ctx), prefix_lens=torch.tensor([128, 0]))
    check(out, lse, ref, torch.float16)


@pytest.mark.parametrize("seqs", [[(5, 70), (9, 9)], [(2, 70), (1, 9)], [(45, 300)]])
def test_rows_outside_every_sequence_stay(cuda_device, device_checks, seqs):
    """A padded batch: rows behind the last sequence hold NaN and infinities, their outputs stay; so
    do rows before the first."""
    from fast_infer_b200.kernels.attention import paged_chunk_attention
    q, k, v, table, cu, ctx = make(seqs, 6, 2, torch.float16)
    n = q.shape[0]
    pad = torch.full((4, 6, D), math.nan, dtype=q.dtype)
    pad[2:] = math.inf
    big = torch.cat([pad, q, pad]).to(cuda_device)
    out = torch.full_like(big, 7.0)
    got, lse = paged_chunk_attention(big, k.to(cuda_device), v.to(cuda_device), table.to(cuda_device), PAGE,
                                     (cu + 4).to(cuda_device), ctx.to(cuda_device), out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr()
    assert (out[:4] == 7.0).all() and (out[4 + n:] == 7.0).all()
    check(out[4:4 + n], lse[4:4 + n], oracle((q, k, v, table, cu, ctx)), torch.float16)


def test_strides(cuda_device, device_checks):
    """q as a slice of a wider projection, caches as one layer of a pool, a strided table and a
    transposed output."""
    from fast_infer_b200.kernels.attention import paged_chunk_attention
    batch = make([(33, 200), (1, 90)], 6, 2, torch.float16)
    q, k, v, table, cu, ctx = (t.to(cuda_device) for t in batch)
    wide = torch.full((q.shape[0], 10, D), 3.0, dtype=q.dtype, device=q.device)
    wide[:, 2:8] = q
    pool = torch.full((2, k.shape[0], PAGE, 4, D), math.nan, dtype=q.dtype, device=q.device)
    pool[1, :, :, 1:3] = k
    table2 = torch.full((table.shape[0], table.shape[1] * 2), -1, dtype=torch.int32, device=q.device)
    table2[:, ::2] = table
    out = torch.empty(6, q.shape[0], D, dtype=q.dtype, device=q.device).transpose(0, 1)
    got, lse = paged_chunk_attention(wide[:, 2:8], pool[1, :, :, 1:3], v, table2[:, ::2], PAGE, cu, ctx,
                                     out=out, return_lse=True)
    check(got, lse, oracle(batch), torch.float16)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=q.device)[1:].view(q.shape)  # unaligned
    odd.copy_(q)
    out = torch.empty(q.numel() + 1, dtype=q.dtype, device=q.device)[1:].view(q.shape)
    got2, _ = paged_chunk_attention(odd, k, v, table.long(), PAGE, cu.long(), ctx.long(), out=out,
                                    return_lse=True)
    assert torch.equal(got2, got)


def test_same_bits_on_other_streams_and_in_graphs(cuda_device):
    """Every run gives the same bits: eager, on a side stream, and a captured graph replayed with new
    lengths and pages in the same buffers."""
    from fast_infer_b200.kernels.attention import paged_chunk_attention
    first = [t.to(cuda_device) for t in make([(40, 333), (1, 700), (90, 200)], 6, 2, torch.float16, 1)]
    second = [t.to(cuda_device) for t in make([(1, 650), (120, 120), (10, 500)], 6, 2, torch.float16, 2)]
    nb = max(first[1].shape[0], second[1].shape[0])
    mb = max(first[3].shape[1], second[3].shape[1])

    def padded(batch):
        q, k, v, table, cu, ctx = batch
        k2, v2 = (torch.zeros(nb, *x.shape[1:], dtype=x.dtype, device=x.device) for x in (k, v))
        k2[:k.shape[0]], v2[:v.shape[0]] = k.nan_to_num(), v.nan_to_num()
        t2 = torch.full((3, mb), -1, dtype=torch.int32, device=q.device)
        t2[:, :table.shape[1]] = table
        return [torch.cat([q, q])[:131].contiguous(), k2, v2, t2, cu, ctx]
    first, second = padded(first), padded(second)

    def call(b):
        out = torch.zeros_like(b[0])
        return paged_chunk_attention(*b[:4], PAGE, *b[4:], return_lse=False, out=out)
    want = [call(first), call(second)]
    assert torch.equal(call(first), want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(second)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[1])
    bufs = [t.clone() for t in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(bufs)
    for b, w in ((second, want[1]), (first, want[0])):
        for x, y in zip(bufs, b):
            x.copy_(y)
        graph.replay()
        assert torch.equal(out, w)


def test_agrees_with_paged_attention(cuda_device, device_checks):
    """Single tokens: the decode kernel's results within both kernels' rounding."""
    from fast_infer_b200.kernels.attention import paged_attention
    batch = make([(1, c) for c in (1, 64, 65, 900, 333)], 24, 8, torch.float16, garbage=0.0)
    q, k, v, table, cu, ctx = (t.to(cuda_device) for t in batch)
    out, lse = run(batch, cuda_device)
    check(out, lse, oracle(batch), torch.float16)
    dec = paged_attention(q, k, v, table, PAGE, 0, context_lens=ctx)
    assert (out.float() - dec.float()).abs().max() <= 2e-3


def test_many_sequences(cuda_device, device_checks):
    """The largest batch one launch takes, and one more."""
    g = torch.Generator().manual_seed(5)
    seqs = [(int(n), int(n) + int(c)) for n, c in zip(torch.randint(0, 3, (2048,), generator=g),
                                                       torch.randint(0, 40, (2048,), generator=g))]
    batch = make(seqs, 2, 1, torch.float16)
    check(*run(batch, cuda_device), oracle(batch), torch.float16)
    with pytest.raises(RuntimeError, match="split the batch"):
        run(make(seqs + [(1, 1)], 2, 1, torch.float16), cuda_device)


@pytest.mark.parametrize("hq,hk,new,ctx", [(4, 1, 8, 8), (4, 1, 7, 300), (6, 2, 150, 400), (8, 8, 20, 20)])
def test_nan_keys_show_where_they_are_seen(cuda_device, device_checks, hq, hk, new, ctx):
    """A NaN key makes NaN of the rows that see it and leaves those before it as they were."""
    batch = make([(new, ctx)], hq, hk, torch.float16)
    bad = new // 2  # a new token
    slot = ctx - new + bad
    batch[1][batch[3][0, slot // PAGE], slot % PAGE] = math.nan
    out, lse = run(batch, cuda_device)
    ref = oracle(batch)  # (takes a NaN key for one that no row sees)
    check(out[:bad], lse[:bad], tuple(x[:bad] for x in ref), torch.float16)
    assert torch.isnan(out[bad:]).all() and torch.isnan(lse[bad:]).all()


@pytest.mark.parametrize("hq,hk,new", [(2, 1, 3), (2, 1, 90)])
def test_distances_at_far_positions(cuda_device, device_checks, hq, hk, new):
    """Past 2^24 positions are not fp32 numbers, but distances within the window are: scores are off
    by the rounding of slope * distance (2^-24 * 2^8 in log2 units) beside what `check` counts."""
    from fast_infer_b200.kernels.attention import attention_mass
    g = torch.Generator().manual_seed(5)
    ctx, window = (1 << 24) + 5003, 200
    k, v = (torch.randn(5, PAGE, hk, D, generator=g).half() for _ in range(2))
    table = torch.randint(0, 5, (1, ctx // PAGE + 1), generator=g).int()
    q = torch.randn(new, hq, D, generator=g).half()
    slopes = torch.tensor([0.5, 0.25])
    # the same keys as a short sequence: pages from the one that holds the first visible key
    first = (ctx - new - window) // PAGE
    short = (q, k, v, table[:, first:], torch.tensor([0, new]).int(),
             torch.tensor([ctx - first * PAGE]).int())
    ref = oracle(short, alibi_slopes=slopes, window=window)
    far = tuple(t.to(cuda_device) for t in
                (q, k, v, table, torch.tensor([0, new]).int(), torch.tensor([ctx]).int()))
    form = dict(alibi_slopes=slopes, window=window)
    out, lse = run(far, cuda_device, **form)
    check(out, lse, ref, torch.float16)
    near = run(short, cuda_device, **form)
    got = attention_mass(far[0], far[1], far[3], PAGE, far[4], far[5], near[1],
                         alibi_slopes=slopes.to(cuda_device), window=window)
    s = tuple(t.to(cuda_device) for t in short)
    want = attention_mass(s[0], s[1], s[3], PAGE, s[4], s[5], near[1],
                          alibi_slopes=slopes.to(cuda_device), window=window)
    n = want.shape[2]
    # (each within 2^-15 relative of the definition: see the tests of attention_mass)
    assert ((got[:, :, first * PAGE:first * PAGE + n] - want).abs() <= want * 2.0 ** -14).all()
    assert not got[:, :, :first * PAGE].any()


@pytest.mark.parametrize("softcap", [1e-3, 1e6])
def test_caps_far_from_the_scores(cuda_device, device_checks, softcap):
    """All scores at the cap's ends, and a cap that changes none."""
    batch = make([(20, 200), (1, 77), (100, 130)], 4, 2, torch.float16)
    check(*run(batch, cuda_device, softcap=softcap), oracle(batch, softcap=softcap), torch.float16)
