"""sample_tokens against the definition in numpy, 64 bits. Tokens are whole numbers and have to be equal: the sums are
held to 2^-45, so a uniform number at random is nowhere near a boundary."""

import math

import numpy as np
import pytest
import torch

from fast_infer_b200.kernels.sampling import sample_tokens

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def kept_set(row, t, k, p, m):
    """Kept indexes, ascending, and all weights, of one row in 64 bits."""
    w = np.exp((row - row.max()) / t)
    order = np.argsort(-row, kind="stable")
    order = order[row[order] > -math.inf]
    if k > 0:
        order = order[:k]
    run = np.concatenate([[0.0], np.cumsum(w[order])])
    keep = run[:-1] < p * run[-1] if p < 1 else np.ones(len(order), bool)
    if m > 0:  # w >= m, as the logarithm has it: exp(-1e-42) is below 1, but not in 64 bits
        keep &= row[order] - row.max() >= t * math.log(m)
    keep[0] = True
    return np.sort(order[keep]), w


def definition(x, u, t, k, p, m):
    out = []
    for r, row in enumerate(x):
        if np.isnan(row).any() or (row == math.inf).any() or not (row > -math.inf).any():
            out.append(-1)
        elif t[r] == 0:
            out.append(int(np.argmax(row)))
        else:
            keep, w = kept_set(row, t[r], k[r], p[r], m[r])
            run = np.cumsum(w[keep])
            out.append(int(keep[min(np.searchsorted(run, u[r] * run[-1], side="right"), len(keep) - 1)]))
    return out


def check(logits, u, t, k, p, m):
    rows, dev = logits.shape[0], logits.device
    args = [torch.as_tensor(np.broadcast_to(np.asarray(a, d), rows).copy()).to(dev)
            for a, d in ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
    got = sample_tokens(logits, u, args[0], top_k=args[1], top_p=args[2], min_p=args[3])
    assert got.dtype == torch.int32 and got.shape == (rows,)
    want = definition(logits.double().cpu().numpy(), u.double().cpu().numpy(),
                      *(a.double().cpu().numpy() if i != 1 else a.cpu().numpy() for i, a in enumerate(args)))
    assert got.tolist() == want
    return got


def draw(dev, rows, vocab, dtype, spread=2.5, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g, device=dev)
    peaks = torch.rand(rows, vocab, generator=g, device=dev) < 8 / vocab
    return (x + 7.0 * peaks).to(dtype), torch.rand(rows, generator=g, device=dev)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.02),
            (1.0, 1, 0.5, 0.5), (1.0, 100000, 0.999, 0.0), (0.05, 0, 0.9, 0.0), (5.0, 3000, 0.3, 0.0), (1.0, 0, 0.01, 0.0),
            (0.0, 7, 0.5, 0.1), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 255, 257, 1000, 4097, 33001, 128256, 151937])
def test_settings(cuda_device, dtype, vocab):
    """Every row with a setting of its own, few rows (a cluster of CTAs each)."""
    rows = 2 * len(SETTINGS)
    x, u = draw(cuda_device, rows, vocab, dtype, seed=vocab)
    check(x, u, *(np.array(SETTINGS * 2).T))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 262144), (3, 262143), (700, 1003), (300, 32000), (170, 65537)])
def test_many_rows_and_the_largest_vocabulary(cuda_device, dtype, rows, vocab):
    x, u = draw(cuda_device, rows, vocab, dtype, seed=rows)
    check(x, u, *(np.resize(np.array(SETTINGS), (rows, 4)).T))


@pytest.mark.parametrize("dtype", TYPES)
def test_ties(cuda_device, dtype):
    """Few distinct values: the cut falls among equals, and the lowest indexes of them stay."""
    g = torch.Generator(device=cuda_device).manual_seed(3)
    for vocab, levels in ((1000, 1), (1000, 3), (40000, 5), (40000, 2)):
        rows = 3 * len(SETTINGS)
        x = torch.randint(0, levels, (rows, vocab), generator=g, device=cuda_device).to(dtype) - 1
        u = torch.rand(rows, generator=g, device=cuda_device)
        check(x, u, *(np.resize(np.array(SETTINGS), (rows, 4)).T))


def test_borders_between_equal_weights(cuda_device):
    """Equal logits: sums are whole, so u and top_p may lie on a border itself. The token is the first whose running
    sum is above u's share; top-p keeps those before which the mass is below its own."""
    x = torch.zeros(9, 1024, device=cuda_device)
    u = torch.tensor([0.0, 1 / 1024, 0.5, 1023 / 1024, 0.25, 0.0, 0.9990234375, 0.5, 0.75], device=cuda_device)
    p = np.array([1.0, 1.0, 1.0, 1.0, 0.5, 0.5, 0.5, 1 / 1024, 0.25])
    got = check(x, u, 1.0, 0, p, 0.0)
    assert got.tolist() == [0, 1, 512, 1023, 128, 0, 511, 0, 192]


@pytest.mark.parametrize("dtype", TYPES)
def test_hidden_and_broken_rows(cuda_device, dtype):
    x, u = draw(cuda_device, 12, 5000, dtype, seed=5)
    x[0, :] = -math.inf                      # nothing left
    x[1, 17] = math.nan
    x[2, 4999] = math.inf
    x[3, 1:] = -math.inf                     # the first alone
    x[4, :-1] = -math.inf                    # the last alone
    x[5, 100:] = -math.inf
    x[6, ::2] = -math.inf
    x[7, :] = torch.finfo(dtype).min         # all of the type's lowest
    x[8, :2500] = torch.finfo(dtype).min
    x[9, 3] = torch.finfo(dtype).max
    x[10, :] = -0.0
    x[10, 1::2] = 0.0                        # equal, whatever the sign
    for setting in SETTINGS:
        got = check(x, u, *setting)
        assert got[:5].tolist() == [-1, -1, -1, 0, 4999]


def test_far_apart_and_tiny_values(cuda_device):
    """Values over the whole range of fp32, subnormal ones among them, whose bits the search goes by."""
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x = torch.randn(26, 3000, generator=g, device=cuda_device)
    x[:13] *= 10.0 ** torch.randint(-44, 38, (13, 3000), generator=g, device=cuda_device).double()
    x[13:] *= 1e-42
    u = torch.rand(26, generator=g, device=cuda_device)
    check(x, u, *(np.array(SETTINGS * 2).T))


def test_scalars_strides_out_and_uniform_edges(cuda_device):
    x, u = draw(cuda_device, 6, 3001, torch.float16, seed=9)
    wide = torch.zeros(6, 4000, dtype=torch.float16, device=cuda_device)
    wide[:, 5:3006] = x
    view = wide[:, 5:3006]                   # rows that begin at any element
    want = sample_tokens(x, u, 0.9, top_k=30, top_p=0.9, min_p=0.01)
    assert torch.equal(sample_tokens(view, u, 0.9, top_k=30, top_p=0.9, min_p=0.01), want)
    out = torch.full((6,), -7, dtype=torch.int32, device=cuda_device)
    assert sample_tokens(x.t().contiguous().t(), u, 0.9, top_k=30, top_p=0.9, min_p=0.01, out=out) is out
    assert torch.equal(out, want)
    assert sample_tokens(x[:0], u[:0]).shape == (0,)
    # the greatest fp32 below 1 finds the last kept token at most
    top = torch.full((6,), 1 - 2.0 ** -24, device=cuda_device)
    check(x, top, 1.0, 0, 1.0, 0.0)
    check(x, torch.zeros(6, device=cuda_device), 1.0, 20, 1.0, 0.0)


def test_same_token_on_every_run_stream_and_replay(cuda_device):
    x, u = draw(cuda_device, 40, 50257, torch.bfloat16, seed=2)
    want = sample_tokens(x, u, 1.0, top_p=0.9)
    for _ in range(5):
        assert torch.equal(sample_tokens(x, u, 1.0, top_p=0.9), want)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        other = sample_tokens(x, u, 1.0, top_p=0.9)
    stream.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_tokens(x, u, 1.0, top_p=0.9)
    x2, u2 = draw(cuda_device, 40, 50257, torch.bfloat16, seed=4)
    want2 = sample_tokens(x2, u2, 1.0, top_p=0.9)
    x.copy_(x2)
    u.copy_(u2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(155, 131064), (150, 131072), (149, 99991)])
def test_long_slices(cuda_device, dtype, rows, vocab):
    """As many tokens a CTA as there can be, in several parts, with and without ties across them."""
    x, u = draw(cuda_device, rows, vocab, dtype, seed=rows)
    x[1::3] = (x[1::3].float() * 2).round().to(dtype) / 2
    x[2::3] = (x[2::3].float() / 4).round().to(dtype)
    check(x, u, *(np.resize(np.array(SETTINGS), (rows, 4)).T))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 150])
def test_many_values_near_zero(cuda_device, dtype, rows):
    """Most logits within many octaves around 0, some of them 0: where the cut lies among them and where it does not."""
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    vocab = 60001
    x = 1e-4 * torch.randn(rows, vocab, generator=g, device=cuda_device)
    x[:, ::50] = 0
    x[:, 7::2000] = 8 + torch.randn(rows, x[:, 7::2000].shape[1], generator=g, device=cuda_device)
    x[1::2, 5::9] -= 3
    check(x.to(dtype), torch.rand(rows, generator=g, device=cuda_device), *(np.resize(np.array(SETTINGS), (rows, 4)).T))
