"""Eviction by attention weight against a sort: which tokens stay (exactly), and that their K, V and
weight move bit for bit, in place and to another pool; ties, NaN, budgets at their edges."""

import math

import pytest
import torch

from oracle.chunk_oracle import evict_keep

pytestmark = pytest.mark.gpu
PAGE, D = 64, 128


def make(lens, layers, heads, dtype=torch.float16, seed=0, cap=None, spare=2):
    g = torch.Generator().manual_seed(seed)
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    nb = sum(pages) + spare
    order = torch.randperm(nb, generator=g).int()
    table = torch.full((len(lens), max(pages + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    k = torch.randn(layers, nb, PAGE, heads, D, generator=g).to(dtype)
    v = torch.randn(layers, nb, PAGE, heads, D, generator=g).to(dtype)
    mass = torch.rand(layers, len(lens), heads, cap or table.shape[1] * PAGE, generator=g) ** 6
    return k, v, table, torch.tensor(lens).int(), mass


def oracle(batch, budget, recent, sinks, out):
    """(kept, mass_out, k_out, v_out) on the CPU; `out` = (k_out, v_out, table) before the call."""
    k, v, table, lens, mass = batch
    k_out, v_out, table_out = out[0].clone(), out[1].clone(), out[2]
    layers, B, heads, _ = mass.shape
    kept = torch.full((layers, B, heads, budget), -1, dtype=torch.int32)
    mass_out = torch.zeros(layers, B, heads, budget)
    for layer in range(layers):
        for b in range(B):
            n = int(lens[b])
            for h in range(heads):
                idx = evict_keep(mass[layer, b, h, :n].tolist(), budget, recent, sinks)
                if not idx:
                    continue
                j = torch.tensor(idx)
                r = torch.arange(len(idx))
                kept[layer, b, h, :len(idx)] = j.int()
                mass_out[layer, b, h, :len(idx)] = mass[layer, b, h, j]
                src, dst = table[b, j // PAGE].long(), table_out[b, r // PAGE].long()
                k_out[layer, dst, r % PAGE, h] = k[layer, src, j % PAGE, h]
                v_out[layer, dst, r % PAGE, h] = v[layer, src, j % PAGE, h]
    return kept, mass_out, k_out, v_out


def same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.int16), b.contiguous().view(torch.int16)) \
        if a.dtype != torch.int32 else torch.equal(a.cpu(), b)


def run_both(batch, dev, budget, recent=0, sinks=0):
    """In place and to another pool, both against the oracle."""
    from fast_infer_b200.kernels.eviction import evict_tokens
    k, v, table, lens, mass = batch
    g = torch.Generator().manual_seed(9)
    per = (budget + PAGE - 1) // PAGE
    B = len(lens)
    table_out = torch.randperm(B * per + 1, generator=g)[:B * per].int().view(B, per)
    pool = torch.full((k.shape[0], B * per + 1, PAGE, k.shape[3], D), 3.0, dtype=k.dtype)
    for out in (None, (pool, -pool, table_out)):
        kd, vd, td, ld, md = (t.to(dev) for t in batch)
        od = None if out is None else tuple(t.to(dev) for t in out)
        kept, mass_out = evict_tokens(kd, vd, td, ld, md, budget, recent=recent, sinks=sinks, out=od)
        ref = oracle(batch, budget, recent, sinks, (k, v, table) if out is None else out)
        assert same(kept, ref[0])
        assert torch.equal(mass_out.cpu().view(torch.int32), ref[1].view(torch.int32))
        ko, vo = (kd, vd) if out is None else od[:2]
        assert same(ko, ref[2]) and same(vo, ref[3])
        assert torch.equal(md.cpu().nan_to_num(), mass.nan_to_num())
        if out is not None:
            assert same(kd, k) and same(vd, v)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,budget,recent,sinks", [
    ([1], 1, 0, 0), ([2], 1, 0, 0), ([2], 1, 1, 0), ([2], 1, 0, 1), ([65], 64, 0, 0),
    ([300, 5, 0, 129, 64], 64, 10, 4), ([700, 333], 200, 50, 3), ([128, 127], 127, 0, 0),
    ([500], 100, 96, 4), ([500], 100, 100, 0), ([500], 100, 0, 100), ([513, 1025], 512, 1, 1)])
def test_budgets(cuda_device, device_checks, lens, budget, recent, sinks, dtype):
    run_both(make(lens, 2, 3, dtype), cuda_device, budget, recent, sinks)


def test_one_head_many_tokens(cuda_device, device_checks):
    run_both(make([9000], 1, 1), cuda_device, 4097, 100, 4)


def test_ties(cuda_device, device_checks):
    """Equal weights everywhere, then few values: the lowest indexes stay."""
    batch = make([400, 90], 1, 2)
    for w in (torch.zeros_like(batch[4]), torch.full_like(batch[4], 0.25), (batch[4] * 4).floor(),
              torch.where(batch[4] > 0.3, 1.0, 1.0 + 2.0 ** -23)):
        run_both(batch[:4] + (w,), cuda_device, 70, 8, 2)


def test_special_weights(cuda_device, device_checks):
    """Infinite, subnormal, NaN and negative weights; NaN and negative count as 0."""
    batch = make([300, 200], 2, 2, seed=3)
    mass = batch[4]
    g = torch.Generator().manual_seed(4)
    pick = torch.randint(0, 8, mass.shape, generator=g)
    for i, w in enumerate((math.inf, math.nan, -1.0, -0.0, 1e-42, -math.inf)):
        mass[pick == i] = w
    run_both(batch[:4] + (mass,), cuda_device, 128, 16, 4)


def test_weights_past_the_length_do_not_count(cuda_device, device_checks):
    batch = make([200, 100], 1, 2)
    batch[4][0, 0, :, 200:] = 100.0
    batch[4][0, 1, :, 100:] = math.nan
    run_both(batch, cuda_device, 80, 4, 4)


def test_long_rows_beyond_shared_memory(cuda_device, device_checks):
    """More tokens than the selection keeps in shared memory (pages shared out over one head)."""
    run_both(make([60000], 1, 1, seed=2), cuda_device, 1000, 64, 4)


def test_missing_pages_are_reported_and_their_tokens_stay_put(cuda_device):
    from fast_infer_b200._runtime import device_checks as checks
    from fast_infer_b200.kernels.eviction import evict_tokens
    batch = make([300], 1, 2)
    batch[2][0, 1] = -1
    k, v, t, n, m = (x.to(cuda_device) for x in batch)
    with checks(True), pytest.raises(RuntimeError, match="page pool"):
        evict_tokens(k, v, t, n, m, 250)
    batch[2][0, 1] = batch[0].shape[1]
    t = batch[2].to(cuda_device)
    with checks(True), pytest.raises(RuntimeError, match="page pool"):
        evict_tokens(k, v, t, n, m, 250)


def test_lengths_past_the_table_are_cut_and_reported(cuda_device):
    from fast_infer_b200._runtime import device_checks as checks
    from fast_infer_b200.kernels.eviction import evict_tokens
    k, v, t, n, m = (x.to(cuda_device) for x in make([128], 1, 2))
    with checks(True), pytest.raises(RuntimeError, match="context length"):
        evict_tokens(k, v, t[:, :2].contiguous(), n + 50, m, 100)


def test_strided_pools_and_graph(cuda_device):
    """Pools with room between heads, and a captured call replayed after its inputs changed."""
    from fast_infer_b200.kernels.eviction import evict_tokens
    batch = make([300, 150], 2, 2)
    k, v, t, n, m = (x.to(cuda_device) for x in batch)
    wide = torch.zeros(2, k.shape[1], PAGE, 5, D, dtype=k.dtype, device=k.device)
    kw, vw = wide[..., :2, :], wide[..., 3:, :]
    kw.copy_(k)
    vw.copy_(v)
    ko, vo = torch.zeros_like(k)[:, :4], torch.zeros_like(v)[:, :4]
    to = torch.arange(4, dtype=torch.int32, device=k.device).view(2, 2)
    graph = torch.cuda.CUDAGraph()
    evict_tokens(kw, vw, t, n, m, 100, recent=5, out=(ko, vo, to))
    with torch.cuda.graph(graph):
        kept, mass_out = evict_tokens(kw, vw, t, n, m, 100, recent=5, out=(ko, vo, to))
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        mass = torch.rand(m.shape, generator=g)
        m.copy_(mass)
        ko.zero_()
        vo.zero_()
        graph.replay()
        ref = oracle(batch[:4] + (mass,), 100, 5, 0, (torch.zeros_like(ko).cpu(),
                                                      torch.zeros_like(vo).cpu(), to.cpu()))
        assert same(kept, ref[0]) and same(ko, ref[2]) and same(vo, ref[3])


def test_cache_evict_bookkeeping(cuda_device, device_checks):
    """KVCache.evict: pages return to the free list, lengths shrink, mass is compacted; the next
    extend takes the freed pages and appends behind the kept tokens."""
    from fast_infer_b200.kv_cache import KVCache
    cache = KVCache(2, 2, D, 640, PAGE, cuda_device, num_blocks=9)
    cu, ctx = cache.extend([300, 70])
    assert cu.tolist() == [0, 300, 370] and ctx.tolist() == [300, 70]
    g = torch.Generator(device=cuda_device).manual_seed(1)
    cache.k.copy_(torch.randn(cache.k.shape, generator=g, device=cuda_device))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g, device=cuda_device))
    before = (cache.k.cpu(), cache.v.cpu(), cache.block_table.cpu())
    mass = torch.rand(2, 2, 2, 640, generator=g, device=cuda_device)
    was = mass.cpu()
    batch = before + (torch.tensor([300, 70]), was)
    ref = oracle(batch, 100, 10, 2, before)
    kept = cache.evict(mass, 100, recent=10, sinks=2)
    assert same(kept, ref[0]) and same(cache.k, ref[2]) and same(cache.v, ref[3])
    assert torch.equal(mass[..., :100].cpu(), ref[1]) and not mass[..., 100:].any()
    assert list(cache.seq_lens) == [100, 70] and len(cache.free_blocks) == 5
    assert (cache.block_table.cpu()[0, 2:] == -1).all()
    assert cache.free_blocks[-3:] == before[2][0, 2:5].tolist()
    with pytest.raises(RuntimeError, match="out of memory"):
        cache.extend([500, 70])
    assert list(cache.seq_lens) == [100, 70] and len(cache.free_blocks) == 5
    with pytest.raises(RuntimeError, match="table full"):
        cache.extend([1000, 0])
    _, ctx = cache.extend([60, 0])
    assert ctx.tolist() == [160, 70] and len(cache.free_blocks) == 4


@pytest.mark.parametrize("budget,recent,sinks", [(70, 8, 2), (200, 0, 4), (1, 0, 0)])
def test_many_rows(cuda_device, device_checks, budget, recent, sinks):
    """Rows enough for selection and move to share a kernel, lengths from none to past the budget."""
    lens = [150, 0, 70, 71, 64, 300, 1, 129, 200, 33] * 4
    run_both(make(lens, 2, 10, seed=7), cuda_device, budget, recent, sinks)


def test_many_rows_with_room_for_more(cuda_device, device_checks):
    """Tables and masses that reach further than any sequence (the most shared memory of a short row)."""
    k, v, table, lens, mass = make([70, 200, 3, 130] * 10, 2, 10, seed=7, cap=8192)
    table = torch.nn.functional.pad(table, (0, 128 - table.shape[1]), value=-1)
    run_both((k, v, table, lens, mass), cuda_device, 65, 8, 2)


def test_many_rows_with_a_missing_page(cuda_device):
    """A token whose page is missing in either table is reported and not moved; the rest is."""
    from fast_infer_b200._runtime import device_checks as checks
    from fast_infer_b200.kernels.eviction import evict_tokens
    k, v, table, lens, mass = make([130] * 40, 2, 10, seed=8)
    table[3, 1] = -1
    out = torch.zeros(2, 40, PAGE, 10, D, dtype=k.dtype)
    table_out = torch.arange(40).int().view(40, 1)
    table_out[5, 0] = 99
    kd, vd, td, ld, md, ko, vo, to = (t.to(cuda_device) for t in
                                      (k, v, table, lens, mass, out, out, table_out))
    with checks(True), pytest.raises(RuntimeError, match="block_table entry"):
        evict_tokens(kd, vd, td, ld, md, 60, out=(ko, vo, to))
    for b in (0, 3, 5, 39):
        for h in (0, 9):
            for r, j in enumerate(evict_keep(mass[1, b, h, :130].tolist(), 60, 0, 0)):
                gone = b == 5 or (b == 3 and PAGE <= j < 2 * PAGE)
                want = torch.zeros(D).half() if gone else k[1, table[b, j // PAGE], j % PAGE, h]
                assert torch.equal(ko[1, b, r, h].cpu(), want)
