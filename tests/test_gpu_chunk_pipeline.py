"""The attention and mass kernels where a CTA has many key tiles of a unit and several units: stages and rings that wrap,
accumulators that are rescaled and used again, score maxima that rise and fall along a sequence; against the definition in
64 bits, and with tolerances that the kernels' own rounding leaves.

Queries and keys are multiples of 1/8 of at most 4, the first dim aside (whole numbers of at most 248 against 4): a score's
128 products are multiples of 2^-6, their sums below 2^13, so that fp32 holds every partial sum exactly, in any order."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE, D, LOG2E = 64, 128, math.log2(math.e)


# ------------------------------------------------------------------------------------ inputs
def flat(j):
    return torch.zeros_like(j)


def rising(j):
    """4.1 log2 units a key tile, 31 tiles up, then from the bottom again."""
    return 8.0 * (j // 128 % 31)


def steep(j):
    """20 log2 units every other tile, twelve up and twelve down."""
    i = j // 256 % 24
    return 20.0 * torch.where(i < 12, i, 23 - i)


def make(dev, seqs, hq, hk, dtype, profile=flat, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    pages = [(c + PAGE - 1) // PAGE for _, c in seqs]
    nb = sum(pages) + 1
    order = torch.randperm(nb, generator=g, device=dev).int()
    table = torch.full((len(seqs), max(pages)), -1, dtype=torch.int32, device=dev)

    def grid(*shape):
        return ((torch.randn(*shape, generator=g, device=dev) * 8).round() / 8).clamp(-4, 4)
    k, v = grid(nb, PAGE, hk, D), torch.randn(nb, PAGE, hk, D, generator=g, device=dev)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
        j = torch.arange(p * PAGE, device=dev).float()
        k[table[b, :p].long(), :, :, 0] = profile(j).view(p, PAGE, 1)
    new = [n for n, _ in seqs]
    q = grid(sum(new), hq, D)
    q[..., 0] = 4.0
    cu = torch.tensor([0] + new, device=dev).cumsum(0).int()
    return q.to(dtype), k.to(dtype), v.to(dtype), table, cu, torch.tensor([c for _, c in seqs], device=dev).int()


# ------------------------------------------------------------------ the definition in 64 bits
def definition(batch, softcap=0.0, alibi_slopes=None, window=0, prefix_lens=None, lse_in=None):
    """o, lse and what their tolerances count: sum p |v|, the sum of |v| that P in fp16 may lose, the greatest argument of
    an exp2; with lse_in the mass and that argument's bound instead."""
    q, k, v, table, cu, ctx = batch
    total, hq, _ = q.shape
    hk = k.shape[2]
    group, dev = hq // hk, q.device
    o, absv, lost = (torch.zeros(total, hq, D, dtype=torch.float64, device=dev) for _ in range(3))
    lse = torch.full((total, hq), -math.inf, dtype=torch.float64, device=dev)
    mass = torch.zeros(len(ctx), hk, table.shape[1] * PAGE, dtype=torch.float64, device=dev)
    top_arg = 0.0
    for b, n in enumerate(ctx.tolist()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        if hi == lo or n == 0:
            continue
        j = torch.arange(n, device=dev)
        pages = table[b, j // PAGE].long()
        back = torch.arange(n - (hi - lo), n, device=dev)[:, None] - j
        see = (back >= 0) & ((back < window) if window else True)
        if prefix_lens is not None:
            see = see | (j < int(prefix_lens[b]))
        for h in range(hk):
            kb, vb = k[pages, j % PAGE, h].double(), v[pages, j % PAGE, h].double()
            rows = q[lo:hi, h * group:(h + 1) * group].double()
            s = torch.einsum("ngd,kd->ngk", rows, kb) * D ** -0.5
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            size = s.abs().amax()
            if alibi_slopes is not None:
                bias = alibi_slopes[h * group:(h + 1) * group, None].double() * back.abs()[:, None]
                size = size + (bias * see[:, None]).amax()
                s = s - bias
            s = s.masked_fill(~see[:, None], -math.inf)
            if lse_in is not None:
                l = lse_in[lo:hi, h * group:(h + 1) * group].double()
                top_arg = max(top_arg, float(size + l.abs().amax()))
                mass[b, h, :n] = torch.exp(s - l[..., None]).sum((0, 1))
                continue
            top_arg = max(top_arg, float(size))
            top = s.amax(-1, keepdim=True)
            e = torch.exp(s - top)
            l = e.sum(-1, keepdim=True)
            heads = slice(h * group, (h + 1) * group)
            o[lo:hi, heads], absv[lo:hi, heads] = e @ vb / l, e @ vb.abs() / l
            lost[lo:hi, heads] = torch.where(e < 2.0 ** -13, e.clamp(max=2.0 ** -25), 0.0) @ vb.abs() / l
            lse[lo:hi, heads] = (top + torch.log(l))[..., 0]
    return (mass, top_arg * LOG2E) if lse_in is not None else (o, lse, absv, lost, top_arg * LOG2E)


# ------------------------------------------------------------ how the launch's work is cut up
def chunk_parts(seqs, hq, hk, window=0, prefix=0, sms=148):
    """The narrow and the wide kernel's work: for every CTA the (sequence, first key tile, last, tiles of the unit) of its
    parts, as the kernels cut their lines."""
    group, batch, total = hq // hk, len(seqs), sum(n for n, _ in seqs)
    per_unit = 32 // group if group <= 32 else 0
    narrow = per_unit > 0 and (batch > 1 or total <= per_unit)
    wide = per_unit == 0 or total > batch * per_unit or total - batch >= 500
    out = []
    for on, is_narrow in ((narrow, True), (wide, False)):
        unit = per_unit if is_narrow else 2 * (128 // group)
        pad = 3 if is_narrow else 2
        units = []
        for b, (n, c) in enumerate(seqs):
            if not on or n == 0 or (narrow and wide and (n * group <= 32) != is_narrow):
                continue
            for t0 in range(0, n, unit):
                p0, p1 = c - n + t0, c - n + min(t0 + unit, n) - 1
                last = (min(c, max(p1 + 1, prefix)) - 1) // 128
                lo = min(max(p0 - window + 1, 0) // 128, last) if window else 0
                units.append((b, min(-(-prefix // 128), lo) + last - lo + 1))
        line = [u for _ in range(hk) for u in units]
        steps = sum(n + pad for _, n in line)
        ctas = [[] for _ in range(min(steps, sms))]
        at = 0
        for b, n in line:
            for c in range(at * len(ctas) // steps, len(ctas)):
                first, end = steps * c // len(ctas), steps * (c + 1) // len(ctas)
                if first >= at + n + pad:
                    break
                j0, j1 = max(first - at - pad, 0), min(end - at, n + pad) - pad
                if j1 > j0:
                    ctas[c].append((b, j0, j1, n))
            at += n + pad
        out.append(ctas)
    return out


def most(ctas):
    """(most key tiles of one part, most parts of one CTA)"""
    return max(j1 - j0 for c in ctas for _, j0, j1, _ in c), max(len(c) for c in ctas)


def mass_steps(seqs, hq, hk, window=0, prefix=0, sms=148):
    """(mean steps of a CTA, most query tiles of a unit): a step is a unit of keys and a query tile that sees any of them."""
    tile, total = 128 // (hq // hk), sum(n for n, _ in seqs)
    keys = 128 * (4 if total > len(seqs) * tile else 2)
    steps = [0]
    for n, c in seqs:
        for k0 in range(0, c, keys):
            lo, hi = 0, n
            if k0 >= prefix:
                lo = max(k0 - (c - n), 0)
                hi = min(n, min(k0 + keys, c) - 1 + window - (c - n)) if window else n
            steps.append((hi - 1) // tile + 1 - lo // tile if lo < hi else 0)
    return sum(steps) * hk / sms, max(steps)


# --------------------------------------------------------------------------------- tolerances
def cap_error(softcap):
    """Of a capped score, in log2 units: tanh to 2^-21 (its argument's rounding, polynomial or exp2, reciprocal)."""
    return softcap * LOG2E * 2.0 ** -21


def check_attention(got, ref, dtype, tiles, softcap=0.0):
    """Relative error E of a weight or of a sum of them: exp2 (2^-22: the hardware's bound; the polynomial has 2.2e-7), its
    use in a rescale, in the merge of two sums and in the join (a rescale shrinks what came before by 2^8 or more, so only
    the last one's error counts, twice at most); roundings of arguments of up to S log2 units (scale, product, bias, max,
    difference, partial lse, its difference: 16 half steps together); sums of 16 values a thread and tile and of the tiles
    (24 + tiles half steps). lse has E and the rounding of itself and ln 2. o has E twice, P's and its own rounding (half a
    step each), 8 accumulations a tile of at most two half steps in 32 bits each, and what fp16 loses of small P."""
    out, lse = got
    o, l, absv, lost, s = ref
    u = torch.finfo(dtype).eps / 2
    e = 5 * 2.0 ** -22 + 16 * 2.0 ** -24 * s + (24 + tiles) * 2.0 ** -24 + cap_error(softcap)
    diff = (lse.double() - l).abs()
    assert (diff <= e + 2.0 ** -22 * l.abs()).all(), f"lse: {float(diff.max()):.3e}, E {e:.3e}"
    tol = u * (absv + o.abs()) * (1 + 2.0 ** -8) + (2 * e + 16 * tiles * 2.0 ** -24) * absv + \
        (2.0 ** -24 + lost if dtype == torch.float16 else 0.0)
    diff = (out.double() - o).abs()
    assert (diff <= tol).all(), f"o: {float((diff - tol).max()):.3e} past the tolerance"


def call(batch, **form):
    from fast_infer_b200.kernels.attention import paged_chunk_attention
    q, k, v, table, cu, ctx = batch
    return paged_chunk_attention(q, k, v, table, PAGE, cu, ctx, return_lse=True, **form)


LONG = [(700, 9700)]
TOKENS = [(1, 4000 - 7 * i) for i in range(64)]
DRAFTS = [(2 + i % 9, 1500 + 131 * i) for i in range(30)]
MIXED = [(1 + (i * 37) % 300, 300 + (i * 577) % 2900) if i % 3 else (1 + i % 7, 500 + 90 * i) for i in range(36)]


def form_of(name, dev, seqs, hq):
    slopes = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev).float() / hq)
    return {"plain": {}, "cap": dict(softcap=30.0), "alibi": dict(alibi_slopes=slopes),
            "cap_alibi": dict(softcap=20.0, alibi_slopes=slopes),
            "window": dict(window=1000, prefix_lens=torch.full((len(seqs),), 300, dtype=torch.int32, device=dev))}[name]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("profile", [flat, rising, steep])
@pytest.mark.parametrize("form", ["plain", "cap", "alibi", "cap_alibi", "window"])
@pytest.mark.parametrize("name", ["long", "tokens", "drafts", "mixed"])
def test_attention(cuda_device, device_checks, name, form, profile, dtype):
    seqs = dict(long=LONG, tokens=TOKENS, drafts=DRAFTS, mixed=MIXED)[name]
    limits = dict(window=1000, prefix=300) if form == "window" else {}
    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    narrow, wide = chunk_parts(seqs, 24, 8, sms=sms, **limits)
    # what these batches are for: every ring wraps, every accumulator is used again
    if name != "long":
        tiles, units = most(narrow)
        assert tiles >= 6 and units >= 2, (tiles, units)
    if name in ("long", "mixed"):
        tiles, units = most(wide)
        assert tiles >= 6 and units >= 2, (tiles, units)
    batch = make(cuda_device, seqs, 24, 8, dtype, profile)
    f = form_of(form, cuda_device, seqs, 24)
    got = call(batch, **f)
    check_attention(got, definition(batch, **f), dtype, max(c for _, c in seqs) // 128 + 2, f.get("softcap", 0.0))
    again = call(batch, **f)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_maxima_rise_within_a_part(cuda_device):
    """The profiles do what they are for: in some CTA's part the greatest score rises past the bound of a rescale, more
    than once, after the tile that sets it (for the narrow kernel: a warpgroup's, every other tile)."""
    step = 4 * D ** -0.5 * LOG2E
    for profile in (rising, steep):
        for seqs, which, stride in ((LONG, 1, 1), (MIXED, 1, 1), (TOKENS, 0, 2), (DRAFTS, 0, 2)):
            moves = 0
            for cta in chunk_parts(seqs, 24, 8)[which]:
                for _, j0, j1, _ in cta:
                    top, count = None, 0
                    for j in range(j0, j1, stride):
                        x = float(profile(torch.tensor([float(j * 128)]))[0]) * step
                        if top is None:
                            top = x
                        elif x > top + 8 + 2:  # (the other dims' share of a maximum varies by less than 2)
                            top, count = x, count + 1
                    moves = max(moves, count)
            assert moves >= 1, (profile.__name__, len(seqs))


@pytest.mark.parametrize("new,hq,hk", [(300, 2, 1), (300, 24, 8), (9, 2, 1)])
def test_exp2_to_its_last_digits(cuda_device, device_checks, new, hq, hk):
    """A window of two keys: lse shows the error of a single exp2, at every column of a tile and any fraction."""
    seqs = [(new, 300 + new)] * 3
    batch = make(cuda_device, seqs, hq, hk, torch.float16)
    got = call(batch, window=2)
    check_attention(got, definition(batch, window=2), torch.float16, 1)


MASS = {"last_tokens": [(300, 30000)], "tokens": TOKENS, "drafts": DRAFTS, "mixed": MIXED, "whole": [(2100, 3000)]}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["plain", "cap", "alibi", "cap_alibi", "window"])
@pytest.mark.parametrize("name", list(MASS))
def test_mass(cuda_device, device_checks, name, form, dtype):
    """Per value: exp2 (2^-22), roundings of an argument whose parts reach S log2 units (lse, scale, bias, sum: 8 half steps),
    32 values summed a thread and step and the steps among each other (40 + steps half steps), the cap's tanh."""
    from fast_infer_b200.kernels.attention import attention_mass
    seqs = MASS[name]
    limits = dict(window=1000, prefix=300) if form == "window" else {}
    mean, deep = mass_steps(seqs, 24, 8, **limits)
    if name != "last_tokens" or form != "window":
        assert mean >= 9  # more than the rings of units (4) and of rows (4) hold
    if name in ("last_tokens", "whole") and form != "window":
        assert deep >= 5
    batch = make(cuda_device, seqs, 24, 8, dtype)
    q, k, _, table, cu, ctx = batch
    f = form_of(form, cuda_device, seqs, 24)
    lse = definition(batch, **f)[1].float()
    want, s = definition(batch, lse_in=lse, **f)
    got = attention_mass(q, k, table, PAGE, cu, ctx, lse, **f)
    rel = 2.0 ** -22 + 8 * 2.0 ** -24 * s + (40 + deep) * 2.0 ** -24 + cap_error(f.get("softcap", 0.0))
    diff = (got.double() - want).abs()
    assert (got[want == 0] == 0).all()
    # each of a key's weights, one a row, that lies below fp32's normal range counts as 0: at most 2^-126 a row
    small = 2.0 ** -126 * max(n for n, _ in seqs) * 3
    assert (diff <= rel * want + small).all(), f"{float((diff / want.clamp(min=1e-30)).max()):.3e}, {rel:.3e}"
    more = attention_mass(q, k, table, PAGE, cu, ctx, lse, mass=got.clone(), **f)
    assert ((more.double() - 2 * got.double()).abs() <= 2.0 ** -24 * 2 * got.double()).all()


@pytest.mark.parametrize("hq", [1, 2, 16, 17])
def test_mass_of_single_rows(cuda_device, device_checks, hq):
    """Few rows: each column's exp2 shows by itself."""
    from fast_infer_b200.kernels.attention import attention_mass
    batch = make(cuda_device, [(1, 5000)], hq, 1, torch.float16)
    q, k, _, table, cu, ctx = batch
    lse = definition(batch)[1].float()
    want, s = definition(batch, lse_in=lse)
    got = attention_mass(q, k, table, PAGE, cu, ctx, lse)
    rel = 2.0 ** -22 + 8 * 2.0 ** -24 * s + 20 * 2.0 ** -24
    assert ((got.double() - want).abs() <= rel * want).all(), float(((got.double() - want).abs() / want).nan_to_num().max())
