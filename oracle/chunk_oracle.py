"""Oracle of the operators over new tokens and a paged cache (TEST INFRASTRUCTURE ONLY):
attention of a chunk, the weight each cached token receives, eviction and rotary positions with
several axes, from their definitions in 64 bits with one loop per sequence and head."""

from __future__ import annotations

import math

import torch


def gather(cache, table_row, n):
    """Tokens [n, heads, D] of a sequence in float64; pages with an invalid entry give NaN."""
    num_blocks = cache.shape[0]
    out = torch.full((n,) + cache.shape[2:], math.nan, dtype=torch.float64)
    for j in range(n):
        page = int(table_row[j // 64])
        if 0 <= page < num_blocks:
            out[j] = cache[page, j % 64].double()
    return out


def scores(q, k, pos, valid, *, scale, softcap=0.0, slope=0.0, window=0, prefix=0):
    """Scores [n, keys] of one head with -inf where a token does not see a key."""
    s = q.double() @ torch.nan_to_num(k).t() * scale
    if softcap > 0:
        s = softcap * torch.tanh(s / softcap)
    p = pos[:, None]
    j = torch.arange(k.shape[0])[None]
    s = s - slope * (p - j).abs().double()
    see = j <= p
    if window > 0:
        see = see & (j > p - window)
    see = (see | (j < prefix)) & valid[None]
    return s.masked_fill(~see, -math.inf)


def chunk(q, k_cache, v_cache, table, cu, ctx, *, scale=128 ** -0.5, softcap=0.0, slopes=None,
          window=0, prefix=None):
    """(o, lse, weight of |v|, largest |q||k| sum) of CPU tensors; the last two bound the error."""
    total, hq, d = q.shape
    hk = k_cache.shape[2]
    o = torch.zeros(total, hq, d, dtype=torch.float64)
    lse = torch.full((total, hq), -math.inf, dtype=torch.float64)
    absv = torch.zeros_like(o)
    for b in range(len(ctx)):
        lo, hi, n = int(cu[b]), int(cu[b + 1]), int(ctx[b])
        keys = max(n, 0)
        k, v = gather(k_cache, table[b], keys), gather(v_cache, table[b], keys)
        valid = ~torch.isnan(k).all(-1).all(-1)
        pos = torch.arange(n - (hi - lo), n)
        for h in range(hq):
            kh = h // (hq // hk)
            s = scores(q[lo:hi, h], k[:, kh], pos, valid, scale=scale, softcap=softcap,
                       slope=float(slopes[h]) if slopes is not None else 0.0, window=window,
                       prefix=int(prefix[b]) if prefix is not None else 0)
            w = torch.nan_to_num(torch.softmax(s, -1))
            x = torch.nan_to_num(v[:, kh])
            o[lo:hi, h] = w @ x
            absv[lo:hi, h] = w @ x.abs()
            lse[lo:hi, h] = torch.logsumexp(s, -1)
    return o, lse, absv


def mass(q, k_cache, table, cu, ctx, lse, *, scale=128 ** -0.5, softcap=0.0, slopes=None, window=0,
         prefix=None):
    """[batch, hk, table span] of CPU tensors, and the rows that each value sums."""
    hq, hk = q.shape[1], k_cache.shape[2]
    out = torch.zeros(len(ctx), hk, table.shape[1] * 64, dtype=torch.float64)
    for b in range(len(ctx)):
        lo, hi, n = int(cu[b]), int(cu[b + 1]), int(ctx[b])
        keys = max(n, 0)
        k = gather(k_cache, table[b], keys)
        valid = ~torch.isnan(k).all(-1).all(-1)
        pos = torch.arange(n - (hi - lo), n)
        for h in range(hq):
            kh = h // (hq // hk)
            s = scores(q[lo:hi, h], k[:, kh], pos, valid, scale=scale, softcap=softcap,
                       slope=float(slopes[h]) if slopes is not None else 0.0, window=window,
                       prefix=int(prefix[b]) if prefix is not None else 0)
            w = torch.exp(s - lse[lo:hi, h].double()[:, None])
            w[s == -math.inf] = 0.0
            out[b, kh, :keys] += w.sum(0)
    return out


def evict_keep(weights, budget, recent, sinks):
    """Old slots that stay of one head's weights (a list of Python floats), ascending."""
    n = len(weights)
    if n <= budget:
        return list(range(n))
    key = [w if w > 0 else 0.0 for w in weights]  # NaN > 0 is false
    middle = sorted(range(sinks, n - recent), key=lambda j: (-key[j], j))
    return sorted(list(range(sinks)) + middle[:budget - sinks - recent] + list(range(n - recent, n)))


def rope_axes(x, positions, sections, cos, sin):
    """Rotate-half RoPE of x [T, H, 128] in float64; frequency f uses its axis's position."""
    out = torch.empty(x.shape, dtype=torch.float64)
    f0 = 0
    for axis, count in enumerate(sections):
        for f in range(f0, f0 + count):
            p = positions[axis].long()
            lo, hi = x[:, :, f].double(), x[:, :, f + 64].double()
            out[:, :, f] = lo * cos[p, f, None].double() - hi * sin[p, f, None].double()
            out[:, :, f + 64] = hi * cos[p, f + 64, None].double() + lo * sin[p, f + 64, None].double()
        f0 += count
    return out
