"""Operators of serving a long context in chunks over a bounded paged cache, and how their cost is measured.

Four operators, in the order in which a serving loop runs them: rotary positions with several
axes and the cache write (``rope``), attention of new tokens over the paged cache (``chunk``), the
attention weight that each cached token received (``mass``), and the eviction of the cache by that
weight (``evict``). ``run`` computes them in plain torch operations, or, where ``own`` is true, by
the framework's calls.

Conventions. Pages hold 64 tokens, heads 128 values. New tokens are packed: sequence b owns rows
[cu[b], cu[b+1]); ctx[b] counts its cached tokens with the new ones, so its i-th new token has
position ctx[b] - n[b] + i, which is its slot as well.
"""

import math
import random

import numpy as np
import torch

own = False

PAGE, D = 64, 128


def listed():
    return [
        # One request, one new token over a short context: the call whose latency a user waits for.
        dict(name="chunk_one_token", op="chunk", dtype="fp16", hq=24, hkv=8, batch=1, new_lo=1, new_hi=1, past_lo=516,
             past_hi=516, softcap=0.0, alibi=False, window=0, prefix=0, lens=1),
        # Drafted tokens verified against the cache for a batch of requests; scores capped.
        dict(name="chunk_verify", op="chunk", dtype="bf16", hq=24, hkv=8, batch=16, new_lo=2, new_hi=6, past_lo=500,
             past_hi=4090, softcap=50.0, alibi=False, window=0, prefix=0, lens=2),
        # A server's mixed step: prompts' chunks and single tokens together, a distance bias, a
        # sliding window and a prefix that every token sees.
        dict(name="chunk_mixed", op="chunk", dtype="fp16", hq=24, hkv=8, batch=24, new_lo=1, new_hi=1500, past_lo=3,
             past_hi=4000, softcap=0.0, alibi=True, window=1024, prefix=197, lens=3),
        # One chunk of a long document's prefill, far into the document.
        dict(name="chunk_long", op="chunk", dtype="fp16", hq=24, hkv=8, batch=1, new_lo=4096, new_hi=4096,
             past_lo=61003, past_hi=61003, softcap=0.0, alibi=False, window=0, prefix=0, lens=4),
        # Weights received during a decode step of a batch.
        dict(name="mass_decode", op="mass", dtype="fp16", hq=24, hkv=8, batch=16, new_lo=1, new_hi=1, past_lo=1000,
             past_hi=4095, softcap=0.0, alibi=False, window=0, prefix=0, lens=5),
        # Weights of the last tokens of long prompts (what an eviction after the prefill looks at).
        dict(name="mass_last_tokens", op="mass", dtype="bf16", hq=24, hkv=8, batch=4, new_lo=64, new_hi=64,
             past_lo=8000, past_hi=16000, softcap=50.0, alibi=False, window=0, prefix=0, lens=6),
        # Weights of a whole chunk of a long prefill.
        dict(name="mass_chunk", op="mass", dtype="fp16", hq=24, hkv=8, batch=1, new_lo=2048, new_hi=2048,
             past_lo=30011, past_hi=30011, softcap=0.0, alibi=False, window=0, prefix=0, lens=7),
        # One layer of one short request: latency.
        dict(name="evict_one_layer", op="evict", dtype="fp16", hkv=8, layers=1, batch=1, past_lo=777, past_hi=777,
             budget=256, recent=32, sinks=4, lens=8),
        # All layers of a batch whose requests have outgrown their share of the pool.
        dict(name="evict_batch", op="evict", dtype="fp16", hkv=8, layers=28, batch=16, past_lo=900, past_hi=4096,
             budget=1024, recent=128, sinks=4, lens=9),
        # All layers of one long prompt, compressed after its prefill.
        dict(name="evict_long", op="evict", dtype="bf16", hkv=8, layers=28, batch=1, past_lo=32768, past_hi=32768,
             budget=8191, recent=64, sinks=4, lens=10),
        # A decode step of sequences whose cache was compressed: positions ahead of the slots.
        dict(name="rope_decode", op="rope", dtype="fp16", hq=24, hkv=8, batch=64, new_lo=1, new_hi=1, past_lo=200,
             past_hi=1023, axes=1, lens=11),
        # Prompts with images: positions of time, height and width.
        dict(name="rope_images", op="rope", dtype="bf16", hq=24, hkv=8, batch=5, new_lo=700, new_hi=4095, past_lo=0,
             past_hi=600, axes=3, lens=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["chunk", "mass", "evict", "rope"])
    case = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), lens=rng.randrange(1 << 30))
    hkv = rng.choice([1, 2, 4, 8])
    if op == "evict":
        top = _log_int(rng, 65, 32768)
        layers = rng.choice([1, 2, 16, 28])
        room = max(1, 28 * 32768 * 8 // (layers * hkv * top))
        budget = _log_int(rng, 16, max(17, top // 2))
        case.update(hkv=hkv, layers=layers, batch=_log_int(rng, 1, min(64, room)), past_lo=max(1, top // 5), past_hi=top,
                    budget=budget, recent=rng.randrange(0, budget // 2 + 1), sinks=rng.choice([0, 1, 4]))
        return case
    case.update(hq=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv)
    if op == "rope":
        batch = _log_int(rng, 1, 128)
        top = _log_int(rng, 1, max(2, 16384 // batch))
        case.update(batch=batch, new_lo=max(1, top // 6), new_hi=top, past_lo=0,
                    past_hi=_log_int(rng, 1, 2000), axes=rng.choice([1, 2, 3]))
        return case
    batch, new, past = _log_int(rng, 1, 64), _log_int(rng, 1, 4096), _log_int(rng, 64, 65536)
    # no dearer than the largest listed case, and the scores of one KV head within 4 GB
    most = min(5_000_000_000 // case["hq"], 1_000_000_000 // (case["hq"] // hkv))
    while batch > 1 and (batch * (past + new) > 260000 or batch * new * (past + new) > most):
        batch = batch // 2
    while new > 1 and batch * new * (past + new) > most:
        new = new // 2
    case.update(batch=batch, new_lo=max(1, new // 8), new_hi=new, past_lo=max(1, past // 8), past_hi=past,
                softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.25,
                window=_log_int(rng, 16, past) if rng.random() < 0.25 else 0,
                prefix=_log_int(rng, 1, past) if rng.random() < 0.25 else 0)
    return case


# ------------------------------------------------------------------------------------- sizes
def _sizes(case):
    """New and cached (with the new) tokens of every sequence; they belong to the case, not to the seed."""
    rng = random.Random(case["lens"])
    lo, hi = case.get("new_lo", 0), case.get("new_hi", 0)
    new = [_log_int(rng, lo, hi) if hi else 0 for _ in range(case["batch"])]
    ctx = [rng.randint(case["past_lo"], case["past_hi"]) + n for n in new]
    return np.array(new, np.int64), np.array(ctx, np.int64)


def _visible_pairs(case):
    """(pairs of a token and a key that it sees, keys that any token of their sequence sees)"""
    new, ctx = _sizes(case)
    pairs = keys = 0
    for n, c in zip(new, ctx):
        pos = np.arange(c - n, c)
        lo = np.maximum(pos - case["window"] + 1, 0) if case["window"] else np.zeros_like(pos)
        pre = min(case["prefix"], int(c))
        pairs += int(np.sum(np.maximum(pos + 1, pre) - np.clip(lo - pre, 0, None)))
        keys += int(c - max(int(lo[0]) - pre, 0))
    return pairs, keys


def work(case):
    new, ctx = _sizes(case)
    hkv, tokens = case["hkv"], int(new.sum())
    if case["op"] == "evict":
        rows = case["layers"] * hkv
        kept = rows * int(np.minimum(ctx, case["budget"]).sum())
        return {"bytes": rows * int(ctx.sum()) * 4 + kept * (2 * 2 * D * 2 + 4 + 4), "flops": rows * int(ctx.sum())}
    hq = case["hq"]
    if case["op"] == "rope":
        values = tokens * (hq + 2 * hkv) * D
        return {"bytes": 2 * values * 2 + tokens * case["axes"] * 4, "flops": 3 * tokens * (hq + hkv) * D}
    pairs, keys = _visible_pairs(case)
    if case["op"] == "mass":
        return {"bytes": tokens * hq * (D * 2 + 4) + keys * hkv * D * 2 + int(ctx.sum()) * hkv * 4,
                "flops": 2 * D * hq * pairs}
    return {"bytes": tokens * hq * (2 * D * 2 + 4) + keys * hkv * 2 * D * 2, "flops": 4 * D * hq * pairs}


# ------------------------------------------------------------------------------------ inputs
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _tables(g, ctx, spare=3):
    """Block table over shuffled pages, -1 past each sequence's last page, and the pool's page count."""
    pages = (ctx + PAGE - 1) // PAGE
    pool = int(pages.sum()) + spare
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(ctx), int(pages.max()) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages.tolist()):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _int32(a):
    return torch.from_numpy(np.asarray(a, np.int32)).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _dtype(case)
    new, ctx = _sizes(case)
    batch, hkv, tokens = len(ctx), case["hkv"], int(new.sum())

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    st = {"case": case}
    st["table"], pool = _tables(g, ctx)
    if case["op"] == "evict":
        layers, budget = case["layers"], case["budget"]
        st["k"], st["v"] = normal(layers, pool, PAGE, hkv, D), normal(layers, pool, PAGE, hkv, D)
        st["lens"] = _int32(ctx)
        # Weights fall off steeply from a few tokens that draw most of them; a share is equal (zero).
        u = torch.rand(layers, batch, hkv, st["table"].shape[1] * PAGE, generator=g, device="cuda")
        st["mass"] = (0.02 / (u + 1e-4)) * (u < 0.9)
        st["table_out"], pool_out = _tables(g, np.minimum(ctx, budget), spare=0)
        st["k_out"] = torch.zeros(layers, pool_out, PAGE, hkv, D, dtype=dt, device="cuda")
        st["v_out"] = torch.zeros_like(st["k_out"])
        return st
    st["cu"], st["ctx"] = _int32(np.concatenate([[0], np.cumsum(new)])), _int32(ctx)
    hq = case["hq"]
    if case["op"] == "rope":
        st["qkv"] = normal(tokens, (hq + 2 * hkv) * D)
        rows = 20000
        freq = 1.0 / (500000.0 ** (torch.arange(0, D, 2, device="cuda").double() / D))
        angle = torch.outer(torch.arange(rows, device="cuda").double(), freq)
        angle = torch.cat([angle, angle], dim=-1)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        st["positions"] = torch.randint(0, rows, (case["axes"], tokens), generator=g, device="cuda", dtype=torch.int32)
        st["sections"] = {1: (64,), 2: (32, 32), 3: (16, 24, 24)}[case["axes"]]
        st["k_cache"] = torch.zeros(pool, PAGE, hkv, D, dtype=dt, device="cuda")
        st["v_cache"] = torch.zeros_like(st["k_cache"])
        return st
    st["q"] = normal(tokens, hq, D)
    st["k_cache"], st["v_cache"] = normal(pool, PAGE, hkv, D), normal(pool, PAGE, hkv, D)
    st["slopes"] = None
    if case["alibi"]:
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda").float() / hq)
    st["prefix"] = None
    if case["prefix"]:
        st["prefix"] = torch.full((batch,), case["prefix"], dtype=torch.int32, device="cuda")
    if case["op"] == "mass":  # what the attention call before it has returned
        st["lse"] = _plain_attention(st)[1]
    return st


# -------------------------------------------------------------------------------- plain forms
def _padded(st):
    """Row indexes of every sequence's new tokens, padded: index [B, N] into the packed rows, which are real, positions."""
    new = (st["cu"][1:] - st["cu"][:-1]).long()
    i = torch.arange(int(_sizes(st["case"])[0].max()), device="cuda")
    real = i < new[:, None]
    index = torch.where(real, st["cu"][:-1].long()[:, None] + i, 0)
    return index, real, (st["ctx"].long() - new)[:, None] + i


def _head_chunks(st):
    """KV heads in runs whose scores stay within 2 GB."""
    case = st["case"]
    new, _ = _sizes(case)
    group = case["hq"] // case["hkv"]
    each = len(new) * int(new.max()) * group * st["table"].shape[1] * PAGE
    step = max(1, min(case["hkv"], (1 << 29) // each))
    return [slice(h, min(h + step, case["hkv"])) for h in range(0, case["hkv"], step)]


def _plain_scores(st, heads, index, real, pos):
    """Masked scores [B, heads, N * group, C] of a run of KV heads, rows token by token."""
    case = st["case"]
    group = case["hq"] // case["hkv"]
    span = st["table"].shape[1] * PAGE
    q = st["q"].view(-1, case["hkv"], group, D)[index][:, :, heads].float()  # [B, N, h, group, D]
    b, n, h = q.shape[:3]
    q = q.permute(0, 2, 1, 3, 4).reshape(b, h, n * group, D)
    k = st["k_cache"][st["table"].clamp(min=0).long(), :, heads].float()  # [B, pages, 64, h, D]
    k = k.reshape(b, span, h, D).permute(0, 2, 3, 1)
    s = torch.matmul(q, k) * D ** -0.5
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    j = torch.arange(span, device="cuda")
    p = pos[:, :, None]
    if case["alibi"]:
        slope = st["slopes"].view(case["hkv"], group)[heads]
        s = (s.view(b, h, n, group, span) - slope[None, :, None, :, None] * (p - j).abs()[:, None, :, None].float()
             ).view(b, h, n * group, span)
    see = j <= p
    if case["window"]:
        see = see & (j > p - case["window"])
    if case["prefix"]:
        see = see | (j < st["prefix"][:, None, None])
    see = see & (j < st["ctx"][:, None, None]) & real[:, :, None]
    return s.view(b, h, n, group, span).masked_fill(~see[:, None, :, None], -math.inf).view(b, h, n * group, span)


def _plain_attention(st):
    case = st["case"]
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    index, real, pos = _padded(st)
    b, n = index.shape
    o = torch.empty(b, n, hkv, group, D, device="cuda")
    lse = torch.empty(b, n, hkv, group, device="cuda")
    for heads in _head_chunks(st):
        s = _plain_scores(st, heads, index, real, pos)
        h = s.shape[1]
        top = s.amax(-1, keepdim=True)
        top = torch.where(top > -math.inf, top, 0.0)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        v = st["v_cache"][st["table"].clamp(min=0).long(), :, heads].float().reshape(b, -1, h, D).permute(0, 2, 1, 3)
        out = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)
        o[:, :, heads] = out.view(b, h, n, group, D).permute(0, 2, 1, 3, 4)
        lse[:, :, heads] = (top + torch.log(total)).view(b, h, n, group).permute(0, 2, 1, 3)
    return o[real].view(-1, case["hq"], D).to(st["q"].dtype), lse[real].view(-1, case["hq"])


def _plain_mass(st):
    case = st["case"]
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    index, real, pos = _padded(st)
    b, n = index.shape
    mass = torch.empty(b, hkv, st["table"].shape[1] * PAGE, device="cuda")
    for heads in _head_chunks(st):
        s = _plain_scores(st, heads, index, real, pos)
        lse = st["lse"].view(-1, hkv, group)[index][:, :, heads].permute(0, 2, 1, 3).reshape(b, s.shape[1], n * group, 1)
        mass[:, heads] = torch.exp(s - lse).sum(2)
    return mass


def _plain_evict(st):
    case = st["case"]
    budget, layers, hkv = case["budget"], case["layers"], case["hkv"]
    mass, lens = st["mass"], st["lens"].long()
    batch, span = lens.numel(), mass.shape[-1]
    n = lens[None, :, None, None]
    j = torch.arange(span, device="cuda").expand(mass.shape)
    forced = (j < case["sinks"]) | (j >= n - case["recent"]) | (n <= budget)
    key = torch.where(j < n, torch.where(forced, math.inf, mass), -1.0)
    first = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    first = torch.nn.functional.pad(first, (0, max(0, budget - span)), value=span)
    first = torch.where(torch.arange(budget, device="cuda") < n, first, span)  # past the last kept token
    kept = torch.sort(first, dim=-1).values
    live = kept < span
    at = torch.where(live, kept, 0)
    mass_out = torch.where(live, mass.gather(-1, at), 0.0)
    b = torch.arange(batch, device="cuda")[None, :, None, None]
    layer = torch.arange(layers, device="cuda")[:, None, None, None]
    head = torch.arange(hkv, device="cuda")[None, None, :, None]
    page = st["table"].long()[b, at // PAGE]
    slot = torch.arange(budget, device="cuda").expand(kept.shape)
    page_out = st["table_out"].long()[b, slot // PAGE]
    src = [x.expand(kept.shape)[live] for x in (layer, page, at % PAGE, head)]
    dst = [x.expand(kept.shape)[live] for x in (layer, page_out, slot % PAGE, head)]
    st["k_out"][tuple(dst)] = st["k"][tuple(src)]
    st["v_out"][tuple(dst)] = st["v"][tuple(src)]
    return torch.where(live, kept, -1).to(torch.int32), mass_out, st["k_out"], st["v_out"]


def _plain_rope(st):
    case = st["case"]
    hq, hkv = case["hq"], case["hkv"]
    x = st["qkv"].float().view(-1, hq + 2 * hkv, D)
    axis = torch.repeat_interleave(torch.arange(case["axes"], device="cuda"), torch.tensor(st["sections"], device="cuda"))
    axis = torch.cat([axis, axis])
    row = st["positions"].long()[axis].t()  # [T, D]
    d = torch.arange(D, device="cuda")
    cos, sin = st["cos"][row, d][:, None], st["sin"][row, d][:, None]
    rot = x[:, :hq + hkv]
    rot = rot * cos + torch.cat([-rot[..., D // 2:], rot[..., :D // 2]], dim=-1) * sin
    index, real, pos = _padded(st)
    b = torch.arange(index.shape[0], device="cuda")[:, None].expand(index.shape)[real]
    pos = pos[real]
    page = st["table"].long()[b, pos // PAGE]
    st["k_cache"][page, pos % PAGE] = rot[:, hq:].to(st["qkv"].dtype)
    st["v_cache"][page, pos % PAGE] = x[:, hq + hkv:].to(st["qkv"].dtype)
    return rot[:, :hq].to(st["qkv"].dtype), st["k_cache"], st["v_cache"]


def run(state):
    st, case = state, state["case"]
    if own:
        return _own(st, case)
    if case["op"] == "chunk":
        return _plain_attention(st)
    if case["op"] == "mass":
        return _plain_mass(st)
    if case["op"] == "evict":
        return _plain_evict(st)
    return _plain_rope(st)


def _own(st, case):
    if case["op"] == "evict":
        from fast_infer_b200.kernels.eviction import evict_tokens
        kept, mass = evict_tokens(st["k"], st["v"], st["table"], st["lens"], st["mass"], case["budget"],
                                  recent=case["recent"], sinks=case["sinks"],
                                  out=(st["k_out"], st["v_out"], st["table_out"]))
        return kept, mass, st["k_out"], st["v_out"]
    if case["op"] == "rope":
        from fast_infer_b200.kernels.rope import rope_axes_store
        q = rope_axes_store(st["qkv"], case["hq"], st["cos"], st["sin"], st["positions"], st["sections"], st["k_cache"],
                            st["v_cache"], st["table"], PAGE, st["cu"], st["ctx"])
        return q, st["k_cache"], st["v_cache"]
    from fast_infer_b200.kernels.attention import attention_mass, paged_chunk_attention
    form = dict(softcap=case["softcap"], alibi_slopes=st["slopes"], window=case["window"], prefix_lens=st["prefix"])
    if case["op"] == "mass":
        return attention_mass(st["q"], st["k_cache"], st["table"], PAGE, st["cu"], st["ctx"], st["lse"], **form)
    return paged_chunk_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], PAGE, st["cu"], st["ctx"],
                                 return_lse=True, **form)


# ------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(st, case)
    if case["op"] == "rope":
        return _exact_rope(st, case)
    new, ctx = _sizes(case)
    if int(new.sum()) * int(ctx.max()) * case["hq"] > 20_000_000_000:
        return None
    hq, hkv = case["hq"], case["hkv"]
    cu = np.concatenate([[0], np.cumsum(new)])
    span = st["table"].shape[1] * PAGE
    o = torch.zeros(int(cu[-1]), hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(int(cu[-1]), hq, dtype=torch.float64, device="cuda")
    mass = torch.zeros(len(ctx), hkv, span, dtype=torch.float64, device="cuda")
    for b, c in enumerate(ctx.tolist()):
        pages = st["table"][b, :(c + PAGE - 1) // PAGE].long()
        rows = slice(int(cu[b]), int(cu[b + 1]))
        back = torch.arange(c - int(new[b]), c, device="cuda")[:, None] - torch.arange(c, device="cuda")[None]
        hidden = back < 0
        if case["window"]:
            hidden |= back >= case["window"]
        if case["prefix"]:
            hidden[:, :case["prefix"]] = False
        for h in range(hkv):
            k = st["k_cache"][pages, :, h].reshape(-1, D)[:c].double()
            v = st["v_cache"][pages, :, h].reshape(-1, D)[:c].double()
            for x in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                s = st["q"][rows, x].double() @ k.t() / math.sqrt(D)
                if case["softcap"]:
                    s = torch.tanh(s / case["softcap"]) * case["softcap"]
                if case["alibi"]:
                    s -= st["slopes"][x].double() * back.abs()
                s[hidden] = -math.inf
                if case["op"] == "mass":
                    mass[b, h, :c] += torch.exp(s - st["lse"][rows, x].double()[:, None]).sum(0)
                else:
                    lse[rows, x] = torch.logsumexp(s, -1)
                    o[rows, x] = torch.softmax(s, -1) @ v
    return mass if case["op"] == "mass" else (o, lse)


def _exact_evict(st, case):
    kept = torch.full((case["layers"], len(st["lens"]), case["hkv"], case["budget"]), -1, dtype=torch.int32, device="cuda")
    mass = torch.zeros(kept.shape, dtype=torch.float64, device="cuda")
    k_out, v_out = st["k_out"].clone(), st["v_out"].clone()
    for b, n in enumerate(st["lens"].tolist()):
        pages, pages_out = st["table"][b].long(), st["table_out"][b].long()
        w = st["mass"][:, b, :, :n].double()
        take = torch.ones(w.shape, dtype=torch.bool, device="cuda")
        if n > case["budget"]:
            first, last = case["sinks"], n - case["recent"]
            want = case["budget"] - case["sinks"] - case["recent"]
            mid = w[..., first:last]
            if want > 0:
                edge = torch.kthvalue(mid, mid.shape[-1] - want + 1, dim=-1, keepdim=True).values
                over, same = mid > edge, mid == edge
                take[..., first:last] = over | (same & (same.cumsum(-1) <= want - over.sum(-1, keepdim=True)))
            else:
                take[..., first:last] = False
        size = min(n, case["budget"])
        idx = take.nonzero()[:, 2].view(case["layers"], case["hkv"], size)
        kept[:, b, :, :size] = idx.to(torch.int32)
        mass[:, b, :, :size] = w.gather(-1, idx)
        slot = torch.arange(size, device="cuda")
        for h in range(case["hkv"]):
            for layer in range(case["layers"]):
                at = idx[layer, h]
                k_out[layer, pages_out[slot // PAGE], slot % PAGE, h] = st["k"][layer, pages[at // PAGE], at % PAGE, h]
                v_out[layer, pages_out[slot // PAGE], slot % PAGE, h] = st["v"][layer, pages[at // PAGE], at % PAGE, h]
    return kept, mass, k_out.double(), v_out.double()


def _exact_rope(st, case):
    hq, hkv, half = case["hq"], case["hkv"], D // 2
    x = st["qkv"].double().view(-1, hq + 2 * hkv, D)
    q = torch.empty(x.shape[0], hq + hkv, D, dtype=torch.float64, device="cuda")
    f = 0
    for axis, count in enumerate(st["sections"]):
        where = st["positions"][axis].long()
        for d in range(f, f + count):
            lo, hi = x[:, :hq + hkv, d], x[:, :hq + hkv, d + half]
            cos, sin = (st[x][where][:, [d, d + half]].double() for x in ("cos", "sin"))
            q[..., d] = lo * cos[:, :1] - hi * sin[:, :1]
            q[..., d + half] = hi * cos[:, 1:] + lo * sin[:, 1:]
        f += count
    k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
    new, ctx = _sizes(case)
    t = 0
    for b, (n, c) in enumerate(zip(new.tolist(), ctx.tolist())):
        at = torch.arange(c - n, c, device="cuda")
        page = st["table"][b].long()[at // PAGE]
        k_cache[page, at % PAGE] = q[t:t + n, hq:]
        v_cache[page, at % PAGE] = x[t:t + n, hq + hkv:]
        t += n
    return q[:, :hq], k_cache, v_cache
