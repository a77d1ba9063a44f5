"""paged_tree_attention against the definition in 64 bits: trees and chains, 16-bit pages and pages of 8-bit codes.

Tolerances, per row, with p the exact weights and V the cached values (code * scale):
* scores are products of 16-bit (or 8-bit, exact) values summed in fp32 over 128 dims, at most 2^-24 * 130 * sum|q k| * scale off,
  and exp2 turns an absolute error d of a score (in log2 units, with 2^-22.5 of its own) into a relative one of p;
* P is rounded to 16 bits, half a step: fp16 2^-12 .. 2^-11 (p of 2^-13 and less loses up to 2^-25 more), bf16 2^-9 .. 2^-8;
* V times its scale is rounded to q's type where codes are spread to tiles, another half step;
* the output is rounded once, half a step.
Added up as absolute values that bounds |o - exact| by (eps_P + eps_V + d) sum p|V| + eps_o |o| + lost."""

import math

import numpy as np
import pytest
import torch

from fast_infer_b200.kernels.attention import paged_chunk_attention, paged_tree_attention
from fast_infer_b200.kernels.drafting import draft_tree

pytestmark = pytest.mark.gpu
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def make(dev, seqs, hq, hk, dtype, kind, seed=0, spread=0, window=0):
    """seqs: (new, context) of each sequence. Pages are shuffled; unused slots and pages hold NaN (16-bit, e4m3, scales)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    new, ctx = [n for n, _ in seqs], [c for _, c in seqs]
    pages = [-(-c // 64) for c in ctx]
    nb = sum(pages) + 2
    order, at = rng.permutation(nb), 0
    table = np.full((len(seqs), max(pages + [1]) + 1), -1, np.int32)
    used = torch.zeros(nb, 64, dtype=torch.bool, device=dev)
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
        for i in range(p):
            used[table[b, i], :min(64, ctx[b] - 64 * i)] = True
    st = dict(table=torch.from_numpy(table).to(dev), ctx=torch.tensor(ctx, dtype=torch.int32, device=dev),
              cu=torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(dev), seqs=seqs)
    st["q"] = torch.randn(sum(new), hq, 128, generator=g, device=dev).to(dtype)
    for x in "kv":
        rows = torch.randn(nb, 64, hk, 128, generator=g, device=dev)
        if kind == "16bit":
            rows[~used] = math.nan
            st[x], st[x + "s"] = rows.to(dtype), None
        else:
            rows = rows * torch.exp(torch.randn(nb, 64, hk, 1, generator=g, device=dev))
            top = rows.abs().amax(-1, keepdim=True)
            code = rows / top * CODES[kind][1]
            code = (code.round() if kind == "int8" else code).to(CODES[kind][0])
            scale = (top / CODES[kind][1])[..., 0]
            scale[~used] = math.nan
            if kind == "e4m3":
                code.view(torch.uint8)[~used] = 0x7f
            st[x], st[x + "s"] = code, scale.transpose(1, 2).contiguous()
    st["parents"], st["mask"], st["depths"] = None, None, None
    if spread:
        par = []
        for n in new:
            i = np.arange(n)
            p = i - 1 - np.floor(rng.random(n) * np.minimum(i, spread)).astype(np.int64)
            p[(i == 0) | (rng.random(n) < 0.05)] = -1
            par.append(p)
        st["parents"] = par
        flat = torch.from_numpy(np.concatenate(par).astype(np.int32)).to(dev)
        st["mask"], st["depths"] = draft_tree(flat, st["cu"], max(new), window=window)
    return st


def visible(st, window, mask=None):
    """Per sequence [new, context] bool."""
    out, row = [], 0
    bits = None
    m = st["mask"] if mask is None else mask
    if m is not None:
        bits = torch.from_numpy((m.cpu().numpy().view(np.uint32)[..., None] >> np.arange(32) & 1).astype(bool)
                                .reshape(m.shape[0], -1))
    for n, c in st["seqs"]:
        past = c - n
        i, j = torch.arange(n)[:, None], torch.arange(c)[None]
        if bits is None:
            see = (j <= past + i) & ((j > past + i - window) if window else True)
        else:
            depth = st["depths"][row:row + n].cpu()[:, None]
            see = (j < past) & ((j > past + depth - window) if window else True)
            see = see.expand(n, c).clone()
            inner = bits[row:row + n, :n]
            see[:, past:past + inner.shape[1]] = inner
        out.append(see)
        row += n
    return out


def definition(st, softcap=0.0, window=0, mask=None, skip_pages=()):
    q, dev = st["q"], st["q"].device
    total, hq, _ = q.shape
    hk = st["k"].shape[2]
    f = {n: torch.zeros(total, hq, 128, dtype=torch.float64, device=dev) for n in ("o", "absv", "lost")}
    lse = torch.full((total, hq), -math.inf, dtype=torch.float64, device=dev)
    err = torch.zeros(total, hq, dtype=torch.float64, device=dev)
    row = 0
    for b, ((n, c), see) in enumerate(zip(st["seqs"], visible(st, window, mask))):
        if n == 0 or c == 0:
            row += n
            continue
        pages = st["table"][b, :-(-c // 64)].long()
        see = see.to(dev)
        held = ((pages >= 0) & (pages < st["k"].shape[0])).repeat_interleave(64)[:c]
        see = see & held
        safe = pages.clamp(0, st["k"].shape[0] - 1)
        for h in range(hq):
            kh = h // (hq // hk)
            kv = []
            for x in "kv":
                r = st[x][safe][:, :, kh].double()
                if st[x + "s"] is not None:
                    r = r * st[x + "s"][safe, kh].double()[..., None]
                kv.append(torch.where(held[:, None], r.reshape(-1, 128)[:c], 0.0))
            k, v = kv
            rows = slice(row, row + n)
            s = q[rows, h].double() @ k.t() / math.sqrt(128)
            size = q[rows, h].double().abs() @ k.abs().t() / math.sqrt(128)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True)
            some = (top > -math.inf)[:, 0]
            e = torch.where(some[:, None], torch.exp(s - torch.where(some[:, None], top, 0.0)), 0.0)
            e = torch.where(see, e, 0.0)
            l = e.sum(-1, keepdim=True).clamp(min=1e-300)
            f["o"][rows, h], f["absv"][rows, h] = e @ v / l, e @ v.abs() / l
            f["lost"][rows, h] = torch.where(e < 2.0 ** -13, e.clamp(max=2.0 ** -25), 0.0) @ v.abs() / l
            lse[rows, h] = torch.where(some, top[:, 0] + torch.log(l[:, 0]), -math.inf)
            # relative error of any p: scores' sums (their sizes), the cap's 2^-22, and exp2 of arguments up to |s| * log2 e
            worst = torch.where(see, size, 0.0).amax(-1)
            err[rows, h] = worst * (130 + 4) * 2.0 ** -24 + (softcap or 0.0) * 2.0 ** -22 + 2.0 ** -22
        row += n
    return f["o"], f["absv"], f["lost"], lse, err


def check(st, kind, dtype, softcap=0.0, window=0, mask=None, **kw):
    m = st["mask"] if mask is None else mask
    o, lse = paged_tree_attention(st["q"], st["k"], st["v"], st["table"], 64, st["cu"], st["ctx"], tree_mask=m,
                                  depths=st["depths"] if window and m is not None else None, k_scale=st["ks"],
                                  v_scale=st["vs"], softcap=softcap, window=window, return_lse=True, **kw)
    exact, absv, lost, exact_lse, err = definition(st, softcap, window, mask)
    eps = torch.finfo(dtype).eps / 2
    tol = (eps * (1 + (kind != "16bit")) * 1.01 + 2 * err[..., None]) * absv + eps * exact.abs() + lost + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    far = (o.double() - exact).abs()
    assert (far <= tol).all(), (far / tol).max()
    assert torch.equal(torch.isinf(lse), torch.isinf(exact_lse))
    live = ~torch.isinf(exact_lse)
    assert ((lse.double() - exact_lse).abs() <= err + 2.0 ** -22 * exact_lse.abs())[live].all()
    return o, lse


SEQS = {
    "one": [(1, 516)],
    "small": [(1, 1), (5, 5), (0, 70), (9, 64), (3, 65), (10, 129), (1, 0)],
    "trees": [(26, 700), (33, 1290), (1, 300), (64, 64), (8, 1025), (17, 250)],
    "large": [(130, 1500), (85, 2000), (300, 300), (43, 999)],
    "long": [(12, 9000), (60, 12001)],
}


@pytest.mark.parametrize("kind", ["16bit", "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(24, 8), (4, 1), (3, 3), (16, 2)])
@pytest.mark.parametrize("name", list(SEQS))
def test_trees(cuda_device, device_checks, name, heads, dtype, kind):
    seqs = [(n, c) for n, c in SEQS[name] if c >= n]
    for softcap, window in ((0.0, 0), (30.0, 100)):
        st = make(cuda_device, seqs, *heads, dtype, kind, seed=len(name), spread=7, window=window)
        check(st, kind, dtype, softcap, window)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", list(SEQS))
def test_chains_over_codes(cuda_device, device_checks, name, dtype, kind):
    seqs = [(n, c) for n, c in SEQS[name] if c >= n]
    for softcap, window in ((0.0, 0), (50.0, 70)):
        check(make(cuda_device, seqs, 6, 2, dtype, kind, seed=3), kind, dtype, softcap, window)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_chain_is_paged_chunk_attention(cuda_device, dtype):
    st = make(cuda_device, SEQS["trees"], 6, 2, dtype, "16bit")
    args = (st["q"], st["k"], st["v"], st["table"], 64, st["cu"], st["ctx"])
    for kw in (dict(), dict(softcap=20.0, window=90)):
        for a, b in zip(paged_tree_attention(*args, return_lse=True, **kw),
                        paged_chunk_attention(*args, return_lse=True, **kw)):
            assert torch.equal(a, b)
    # and so is the mask of a chain, up to the order of the tiles
    par = torch.cat([torch.arange(n, device=cuda_device) - 1 for n, _ in SEQS["trees"]]).int()
    st["mask"], st["depths"] = draft_tree(par, st["cu"], 64)
    check(st, "16bit", dtype)


@pytest.mark.parametrize("kind", ["16bit", "int8", "e4m3"])
def test_any_mask_and_rows_that_see_nothing(cuda_device, device_checks, kind):
    """Masks of any bits: rows without one (and no cached tokens before) give zeros and -inf; bits past the new tokens
    and past the mask's words count for nothing."""
    dev = cuda_device
    seqs = [(40, 40), (7, 7), (100, 160), (33, 33), (2, 130)]
    st = make(dev, seqs, 6, 2, torch.float16, kind, seed=8, spread=3)
    total = sum(n for n, _ in seqs)
    g = torch.Generator(device=dev).manual_seed(1)
    for words in (1, 4, 5):
        mask = torch.randint(-2 ** 31, 2 ** 31, (total, words), generator=g, device=dev).int()
        mask[::3] = 0
        o, lse = check(st, kind, torch.float16, mask=mask)
        assert (o[0] == 0).all() and torch.isinf(lse[0]).all()


@pytest.mark.parametrize("kind", ["16bit", "int8", "e4m3"])
def test_bad_pages_are_skipped(cuda_device, kind):
    st = make(cuda_device, [(20, 700), (5, 400), (90, 500)], 6, 2, torch.float16, kind, seed=5, spread=4)
    st["table"][0, 3] = -1
    st["table"][1, 0] = 10 ** 6
    st["table"][2, 6] = -7
    check(st, kind, torch.float16)
    from fast_infer_b200._runtime import device_checks
    with device_checks(True), pytest.raises(RuntimeError, match="page pool"):
        paged_tree_attention(st["q"], st["k"], st["v"], st["table"], 64, st["cu"], st["ctx"], tree_mask=st["mask"],
                             k_scale=st["ks"], v_scale=st["vs"])


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_scales_far_apart(cuda_device, device_checks, kind):
    """Rows of zeros (scale 0), and V rows 10^4 apart in size: the small ones still count where they have the weight."""
    st = make(cuda_device, [(3, 500), (30, 300)], 6, 2, torch.bfloat16, kind, seed=6, spread=4)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    st["vs"] *= 10.0 ** (4 * torch.rand(st["vs"].shape, generator=g, device=cuda_device) - 4)
    st["ks"][:, :, ::5] = 0
    st["vs"][:, :, 3::7] = 0
    used = ~torch.isnan(st["vs"])
    assert used.any()
    check(st, kind, torch.bfloat16)


@pytest.mark.parametrize("kind", ["16bit", "int8"])
def test_strides_out_workspace_and_other_stream(cuda_device, device_checks, kind):
    dev = cuda_device
    st = make(dev, SEQS["trees"], 6, 2, torch.float16, kind, seed=9, spread=5)
    o, lse = check(st, kind, torch.float16)
    total = o.shape[0]
    wide = torch.zeros(total + 4, 9, 256, dtype=torch.float16, device=dev)
    q = wide[2:total + 2, 2:8, 128:]
    q.copy_(st["q"])
    both = torch.zeros(2, *st["k"].shape[::-1], device=dev).to(st["k"].dtype)  # heads and slots the other way round
    k, v = (both[i].permute(3, 2, 1, 0) for i in range(2))
    pool = torch.zeros(2, st["k"].shape[2], st["k"].shape[0], 64, 128, device=dev).to(st["k"].dtype)
    k, v = (pool[i].permute(1, 2, 0, 3) for i in range(2))
    k.copy_(st["k"])
    v.copy_(st["v"])
    scales = {}
    if kind == "int8":
        sc = torch.zeros(64, st["ks"].shape[1], st["ks"].shape[0], 2, device=dev)
        scales = dict(k_scale=sc[..., 0].permute(2, 1, 0), v_scale=sc[..., 1].permute(2, 1, 0))
        scales["k_scale"].copy_(st["ks"])
        scales["v_scale"].copy_(st["vs"])
    out = torch.full((total, 9, 128), 7.0, dtype=torch.float16, device=dev)[:, 1:7]
    from fast_infer_b200.kernels.attention import paged_tree_workspace_bytes
    ws = torch.empty(paged_tree_workspace_bytes(total, 6, 2), dtype=torch.uint8, device=dev)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        got = paged_tree_attention(q, k, v, st["table"], 64, st["cu"], st["ctx"], tree_mask=st["mask"], out=out,
                                   workspace=ws, **scales)
    stream.synchronize()
    assert got is out and torch.equal(out, o)


def test_captured_and_replayed(cuda_device):
    """Two graphs, each with a workspace of its own, replayed with lengths and trees that change between replays."""
    dev = cuda_device
    for kind in ("16bit", "int8"):
        a = make(dev, [(20, 700), (4, 90)], 6, 2, torch.float16, kind, seed=1, spread=4)
        b = make(dev, [(12, 650), (12, 80)], 6, 2, torch.float16, kind, seed=2, spread=2)
        graph = torch.cuda.CUDAGraph()
        live = {x: (None if a[x] is None else a[x].clone()) for x in ("q", "mask", "cu", "ctx")}

        def call():
            return paged_tree_attention(live["q"], a["k"], a["v"], a["table"], 64, live["cu"], live["ctx"],
                                        tree_mask=live["mask"], k_scale=a["ks"], v_scale=a["vs"], return_lse=True)
        want_a = call()
        with torch.cuda.graph(graph):
            got = call()
        for x in ("q", "mask", "cu"):
            live[x].copy_(b[x])
        live["ctx"].copy_(torch.tensor([650, 80]))
        want_b = call()
        graph.replay()
        for x, y in zip(got, want_b):
            assert torch.equal(x, y)
        for x in ("q", "mask", "cu", "ctx"):
            live[x].copy_(a[x])
        graph.replay()
        for x, y in zip(got, want_a):
            assert torch.equal(x, y)


def test_nan_scales_show(cuda_device):
    """A cached row that held NaN (scale NaN) makes NaN of the rows that see its key, and of no other's lse."""
    st = make(cuda_device, [(3, 200), (3, 200)], 6, 2, torch.float16, "int8", seed=4)
    page = int(st["table"][0, 1])
    st["ks"][page, 0, 9] = math.nan
    o, lse = paged_tree_attention(st["q"], st["k"], st["v"], st["table"], 64, st["cu"], st["ctx"], k_scale=st["ks"],
                                  v_scale=st["vs"], return_lse=True)
    assert torch.isnan(lse[:3, :3]).all() and torch.isnan(o[:3, :3]).all()
    assert torch.isfinite(lse[:3, 3:]).all() and torch.isfinite(lse[3:]).all() and torch.isfinite(o[3:]).all()


@pytest.mark.parametrize("kind", ["16bit", "int8", "e4m3"])
@pytest.mark.parametrize("seqs", [[(1, 516)], [(1, 300)] * 40, [(60, 3000)], [(1, 9000), (50, 900)]])
def test_workspace_is_as_large_as_what_is_written(cuda_device, device_checks, kind, seqs):
    """The bytes behind the workspace that the sizes ask for stay as they were."""
    from fast_infer_b200.kernels.attention import paged_tree_workspace_bytes
    st = make(cuda_device, seqs, 6, 2, torch.float16, kind, seed=7, spread=3)
    need = paged_tree_workspace_bytes(st["q"].shape[0], 6, 2)
    ws = torch.full((need + (64 << 20),), 171, dtype=torch.uint8, device=cuda_device)
    check(st, kind, torch.float16, workspace=ws[:need])
    assert (ws[need:] == 171).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seqs", [[(1, 300), (8, 200)], [(60, 500)], [(130, 700)]])
def test_every_code(cuda_device, device_checks, seqs, dtype, kind):
    """All bytes that are numbers, -128 of int8 among them, with scales that make scores of a few units."""
    st = make(cuda_device, seqs, 6, 2, dtype, kind, seed=12, spread=4)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    for x in "kv":
        code = torch.randint(-128, 128, st[x].shape, generator=g, device=cuda_device, dtype=torch.int8)
        if kind == "e4m3":
            code = torch.where((code & 0x7f) == 0x7f, 0, code)
        st[x].view(torch.int8).copy_(code)
        st[x + "s"].clamp_(max=2.0 / CODES[kind][1])
    check(st, kind, dtype)


def test_two_streams_at_once(cuda_device):
    """Calls on two streams, each with its own workspace, give what they give alone."""
    dev = cuda_device
    cases = [make(dev, [(60, 6000), (1, 3000)], 6, 2, torch.float16, k, seed=s, spread=4) for k, s in (("int8", 1), ("16bit", 2))]

    def call(st):
        return paged_tree_attention(st["q"], st["k"], st["v"], st["table"], 64, st["cu"], st["ctx"], tree_mask=st["mask"],
                                    k_scale=st["ks"], v_scale=st["vs"])
    want = [call(st) for st in cases]
    streams = [torch.cuda.Stream(dev) for _ in cases]
    torch.cuda.synchronize(dev)
    got = [[], []]
    for _ in range(20):
        for st, stream, out in zip(cases, streams, got):
            with torch.cuda.stream(stream):
                out.append(call(st))
    torch.cuda.synchronize(dev)
    for w, out in zip(want, got):
        assert all(torch.equal(w, o) for o in out)
