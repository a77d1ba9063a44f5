"""Draft trees, acceptance and the move of accepted K and V against plain Python walks. All results are
whole numbers or copies, so they have to be equal."""

import numpy as np
import pytest
import torch

from fast_infer_b200.kernels.drafting import accept_drafts, draft_tree, keep_accepted

pytestmark = pytest.mark.gpu


def trees(rng, sizes, spread, roots=0.05):
    out = []
    for n in sizes:
        i = np.arange(n)
        par = i - 1 - np.floor(rng.random(n) * np.minimum(i, spread)).astype(np.int64)
        par[(rng.random(n) < roots) | (i == 0)] = -1
        out.append(par)
    return out


def packed(parts, dev):
    return torch.from_numpy(np.concatenate([np.zeros(0, np.int64), *parts]).astype(np.int32)).to(dev)


def cu_of(sizes, dev):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).to(dev)


def chain_of(par, i):
    chain = [i]
    while 0 <= par[chain[-1]] < chain[-1]:
        chain.append(int(par[chain[-1]]))
    return chain


def bits_of(mask):
    return (mask.cpu().numpy().view(np.uint32)[..., None] >> np.arange(32) & 1).reshape(mask.shape[0], -1)


@pytest.mark.parametrize("sizes,spread,max_new,window", [
    ([1], 1, 1, 0), ([26], 12, 26, 0), ([0, 33, 0, 64, 1, 31, 32], 8, 64, 0), ([129, 5, 300], 40, 300, 0),
    ([70, 200], 1, 200, 9), ([64, 40], 3, 200, 1), ([4500], 1, 4500, 0), ([4100, 7], 700, 4200, 3)])
def test_draft_tree(cuda_device, device_checks, sizes, spread, max_new, window):
    rng = np.random.default_rng(sum(sizes) + window)
    par = trees(rng, sizes, spread)
    mask, depths = draft_tree(packed(par, cuda_device), cu_of(sizes, cuda_device), max_new, window=window)
    assert mask.shape == (sum(sizes), -(-max_new // 32)) and mask.dtype == torch.int32
    bits, row = bits_of(mask), 0
    for p in par:
        for i in range(len(p)):
            chain = chain_of(p, i)
            want = np.zeros(bits.shape[1], np.int64)
            want[chain[:window or None]] = 1
            assert np.array_equal(bits[row], want) and depths[row].item() == len(chain) - 1, (row, i)
            row += 1


def test_draft_tree_bad_parents_and_rows_outside(cuda_device):
    """A parent that is not below its child makes a root; rows of no sequence stay; a mask that is too short is reported."""
    par = torch.tensor([5, 0, 7, 2, -9, 4, 4, 99, 99], dtype=torch.int32, device=cuda_device)
    cu = torch.tensor([1, 7], dtype=torch.int32, device=cuda_device)
    mask, depths = draft_tree(par, cu, 6)
    # the six nodes' parents: 0 (itself), 7 (past the end), 2 (itself), -9, 4 (itself), 4
    assert depths[1:7].tolist() == [0, 0, 0, 0, 0, 1]
    assert mask[1:7, 0].tolist() == [1, 2, 4, 8, 16, 32 + 16]
    from fast_infer_b200._runtime import device_checks
    with device_checks(True), pytest.raises(RuntimeError, match="context length"):
        draft_tree(torch.full((40,), -1, dtype=torch.int32, device=cuda_device),
                   torch.tensor([0, 40], dtype=torch.int32, device=cuda_device), 32)
    with device_checks(True), pytest.raises(RuntimeError, match="context length"):
        draft_tree(par, torch.tensor([0, 12], dtype=torch.int32, device=cuda_device), 32)


def walk(tokens, sampled, par):
    if len(par) == 0:
        return [], -1
    nodes = [0]
    while True:
        child = [i for i in range(len(par)) if par[i] == nodes[-1] and i > nodes[-1] and tokens[i] == sampled[nodes[-1]]]
        if not child:
            return nodes, int(sampled[nodes[-1]])
        nodes.append(child[0])


@pytest.mark.parametrize("sizes,spread,vocab", [([1], 1, 2), ([26], 4, 2), ([0, 5, 64, 0, 33, 1, 200, 97], 3, 2),
                                                ([31] * 70, 6, 3), ([400, 32], 1, 1), ([40, 40], 40, 1)])
def test_accept_and_keep(cuda_device, device_checks, sizes, spread, vocab):
    """Small vocabularies, so that paths are long and siblings often equal."""
    dev = cuda_device
    for seed in range(3):
        rng = np.random.default_rng(seed + 10 * sum(sizes))
        par = trees(rng, sizes, spread)
        tok = [rng.integers(0, vocab, n) for n in sizes]
        smp = [rng.integers(0, vocab, n) for n in sizes]
        cu = cu_of(sizes, dev)
        path, counts, follow = accept_drafts(packed(tok, dev), packed(smp, dev), packed(par, dev), cu)
        want_path, nodes = [], []
        for b, n in enumerate(sizes):
            p, nxt = walk(tok[b], smp[b], par[b])
            nodes.append(p)
            want_path += p + [-1] * (n - len(p))
            assert counts[b].item() == len(p) and follow[b].item() == nxt
        assert path.tolist() == want_path
        # the move, for every type of a pool
        past = rng.integers(0, 130, len(sizes))
        pages = [-(-(int(p) + n) // 64) for p, n in zip(past, sizes)]
        nb, layers, heads = sum(pages) + 2, 3, 3
        order = rng.permutation(nb)
        table = np.full((len(sizes), max(pages) + 1), -1, np.int32)
        at = 0
        for b, p in enumerate(pages):
            table[b, :p] = order[at:at + p]
            at += p
        bt = torch.from_numpy(table).to(dev)
        ctx = torch.tensor([int(p) + n for p, n in zip(past, sizes)], dtype=torch.int32, device=dev)
        for dtype in (torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn):
            coded = dtype in (torch.int8, torch.float8_e4m3fn)
            raw = [torch.randint(-30000, 30000, (layers, nb, 64, heads, 128), device=dev).to(torch.int16) for _ in "kv"]
            k, v = (r.to(torch.int8).view(dtype) if coded else r.view(dtype) for r in raw)
            ks, vs = (torch.randn(layers, nb, heads, 64, device=dev) for _ in "kv") if coded else (None, None)
            want = [x.clone() for x in (k, v)] + ([x.clone() for x in (ks, vs)] if coded else [])
            for b, p in enumerate(nodes):
                for d, node in enumerate(p):
                    src, dst = int(past[b]) + node, int(past[b]) + d
                    for i, x in enumerate(want):
                        sp, dp = int(table[b, src // 64]), int(table[b, dst // 64])
                        if i < 2:
                            x = x.view(torch.int8) if coded else x.view(torch.int16)
                            x[:, dp, dst % 64] = x[:, sp, src % 64].clone()
                        else:
                            x[:, dp, :, dst % 64] = x[:, sp, :, src % 64].clone()
            keep_accepted(k, v, bt, 64, cu, ctx, path, counts, k_scale=ks, v_scale=vs)
            for got, exp in zip((k, v) + ((ks, vs) if coded else ()), want):
                as_int = torch.int8 if got.dtype in (torch.int8, torch.float8_e4m3fn) else got.dtype
                as_int = torch.int16 if got.dtype in (torch.float16, torch.bfloat16) else as_int
                assert torch.equal(got.view(as_int), exp.view(as_int))


def test_keep_long_path_and_strides(cuda_device, device_checks):
    """More moves than are looked up at a time; pools that are views of larger ones, with heads outermost in memory."""
    dev, n, past = cuda_device, 300, 50
    path = torch.arange(0, n, 2, dtype=torch.int32, device=dev)
    counts = torch.tensor([len(path)], dtype=torch.int32, device=dev)
    path = torch.cat([path, torch.full((n - len(path),), -1, dtype=torch.int32, device=dev)])
    nb = 8
    base = torch.randn(2, 3, nb, 64, 256, device=dev).half()
    k = base[:, :, :, :, :128].permute(0, 2, 3, 1, 4)  # [layers, nb, 64, heads, 128]
    v = base[:, :, :, :, 128:].permute(0, 2, 3, 1, 4)
    bt = torch.randperm(nb, device=dev).int()[None, :6]
    flat = k[:, bt[0].long()].reshape(2, -1, 3, 128).clone(), v[:, bt[0].long()].reshape(2, -1, 3, 128).clone()
    keep_accepted(k, v, bt, 64, torch.tensor([0, n], dtype=torch.int32, device=dev),
                  torch.tensor([past + n], dtype=torch.int32, device=dev), path, counts)
    for x, was in ((k, flat[0]), (v, flat[1])):
        now = x[:, bt[0].long()].reshape(2, -1, 3, 128)
        c = len(range(0, n, 2))
        assert torch.equal(now[:, past:past + c], was[:, past:past + n:2])
        assert torch.equal(now[:, :past], was[:, :past]) and torch.equal(now[:, past + c:], was[:, past + c:])


def test_keep_missing_pages(cuda_device):
    """A token whose page is missing is not moved, and device checks say so; counts and nodes out of range move nothing."""
    dev = cuda_device
    k = torch.randn(1, 4, 64, 1, 128, device=dev).half()
    v = torch.randn(1, 4, 64, 1, 128, device=dev).half()
    was = k.clone(), v.clone()
    cu = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    path = torch.tensor([0, 3, -1, -1], dtype=torch.int32, device=dev)
    counts = torch.tensor([2], dtype=torch.int32, device=dev)
    from fast_infer_b200._runtime import device_checks
    for table, ctx in (([[1, 9]], 66), ([[1, -1]], 66), ([[1, 2]], 2000), ([[1, 2]], 2)):
        bt = torch.tensor(table, dtype=torch.int32, device=dev)
        args = (k, v, bt, 64, cu, torch.tensor([ctx], dtype=torch.int32, device=dev))
        with device_checks(True), pytest.raises(RuntimeError, match="page pool"):
            keep_accepted(*args, path, counts)
    bt = torch.tensor([[1, 2]], dtype=torch.int32, device=dev)
    ctx = torch.tensor([66], dtype=torch.int32, device=dev)
    for bad_path, c in (([0, 9, -1, -1], 2), ([0, -5, 1, -1], 3), ([0, 1, 2, 3], 70), ([0, 3, 2, 1], -3)):
        keep_accepted(k, v, bt, 64, cu, ctx, torch.tensor(bad_path, dtype=torch.int32, device=dev),
                      torch.tensor([c], dtype=torch.int32, device=dev))
    assert torch.equal(k, was[0]) and torch.equal(v, was[1])


def test_other_stream_and_graph(cuda_device):
    """On a stream of their own, and captured and replayed with new inputs."""
    dev = cuda_device
    par = torch.tensor([-1, 0, 0, 1, 2], dtype=torch.int32, device=dev)
    tok = torch.tensor([9, 1, 2, 3, 4], dtype=torch.int32, device=dev)
    smp = torch.tensor([2, 0, 4, 0, 7], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        path, counts, follow = accept_drafts(tok, smp, par, cu)
    stream.synchronize()
    assert (path.tolist(), counts.tolist(), follow.tolist()) == ([0, 2, 4, -1, -1], [3], [7])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        path, counts, follow = accept_drafts(tok, smp, par, cu)
        mask, depths = draft_tree(par, cu, 5)
    smp[0] = 1
    smp[1] = 3
    graph.replay()
    torch.cuda.synchronize()
    assert (path.tolist(), counts.tolist(), follow.tolist()) == ([0, 1, 3, -1, -1], [3], [0])
    assert mask[:, 0].tolist() == [1, 3, 5, 11, 21] and depths.tolist() == [0, 1, 1, 2, 2]
