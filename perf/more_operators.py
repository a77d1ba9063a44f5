"""Operators of serving with drafted tokens over a paged cache of 8-bit values, and how their cost is measured.

Five operators, which one step of such a server runs in this order: the shape of the draft trees as
ancestor masks (``tree``), rotary positions with the write of K and V as 8-bit codes and their reading
back (``cache8``), attention of the drafted tokens over the cache (``attend``), sampling of a token
after each of them (``sample``), and the acceptance of drafts with the move of their K and V
(``accept``). ``run`` computes them in plain torch operations, or, where ``own`` is true, by the
framework's calls.

Conventions. Pages hold 64 tokens, heads 128 values. New tokens are packed: sequence b owns rows
[cu[b], cu[b+1]); ctx[b] counts its cached tokens with the new ones, so its i-th new token has slot
ctx[b] - n[b] + i. Node i of a draft tree is new token i, node 0 the root; parents[i] < i is its
parent's number within the sequence, -1 for a root. Its position is ctx[b] - n[b] + depth.

8-bit values: a row of 128 (one token, one head) has the scale max|x| / Q with Q = 127 (int8) or 448
(e4m3); its codes are Q * x / max|x|, rounded to the nearest code, ties to even.
"""

import math
import random

import numpy as np
import torch

own = False

PAGE, D = 64, 128
Q = {"int8": 127.0, "e4m3": 448.0}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # The new token of one request: latency.
        dict(name="cache8_one_token", op="cache8", dtype="fp16", cache="int8", hq=24, hkv=8, batch=1, new_lo=1, new_hi=1,
             past_lo=516, past_hi=516, lens=1),
        # Prompts of several requests, written to the cache and handed on in 16 bits.
        dict(name="cache8_prompts", op="cache8", dtype="bf16", cache="e4m3", hq=24, hkv=8, batch=5, new_lo=700, new_hi=4095,
             past_lo=0, past_hi=600, lens=12),
        # The tree of one request, as a drafting model has left it on the device.
        dict(name="tree_one", op="tree", batch=1, new_lo=26, new_hi=26, spread=12, window=0, lens=2),
        # Large trees of a full batch, for a layer with a sliding window as well.
        dict(name="tree_batch", op="tree", batch=256, new_lo=40, new_hi=250, spread=40, window=9, lens=3),
        # One request, one new token over a short context: the call whose latency a user waits for.
        dict(name="attend_one_token", op="attend", dtype="fp16", cache="int8", hq=24, hkv=8, batch=1, new_lo=1, new_hi=1,
             past_lo=516, past_hi=516, spread=0, softcap=0.0, window=0, lens=4),
        # A decode step of a batch with long contexts.
        dict(name="attend_decode", op="attend", dtype="bf16", cache="e4m3", hq=24, hkv=8, batch=64, new_lo=1, new_hi=1,
             past_lo=3000, past_hi=9000, spread=0, softcap=0.0, window=0, lens=5),
        # Draft trees verified for a batch over a 16-bit cache; scores capped.
        dict(name="attend_trees_16bit", op="attend", dtype="fp16", cache="16bit", hq=24, hkv=8, batch=16, new_lo=9,
             new_hi=33, past_lo=500, past_hi=4090, spread=8, softcap=50.0, window=0, lens=6),
        # Large trees over long contexts of 8-bit values.
        dict(name="attend_trees_long", op="attend", dtype="bf16", cache="int8", hq=24, hkv=8, batch=8, new_lo=50, new_hi=85,
             past_lo=20000, past_hi=32000, spread=20, softcap=0.0, window=0, lens=7),
        # The next token of one request.
        dict(name="sample_one", op="sample", dtype="fp32", rows=1, vocab=128256, temperature=0.8, top_k=50, top_p=0.9,
             min_p=0.02, lens=8),
        # A token after every node of a batch's trees, rows with settings of their own.
        dict(name="sample_nodes", op="sample", dtype="bf16", rows=253, vocab=128256, temperature=1.0, top_k=0, top_p=0.95,
             min_p=0.0, lens=9),
        # Acceptance for one request, all layers: latency.
        dict(name="accept_one", op="accept", dtype="fp16", hkv=8, layers=28, batch=1, new_lo=26, new_hi=26, past_lo=500,
             past_hi=500, spread=12, lens=10),
        # Acceptance for a batch, all layers.
        dict(name="accept_batch", op="accept", dtype="bf16", hkv=8, layers=28, batch=48, new_lo=20, new_hi=64, past_lo=30,
             past_hi=250, spread=20, lens=11),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache8", "tree", "attend", "attend", "sample", "accept"])
    case = dict(op=op, lens=rng.randrange(1 << 30))
    hkv = rng.choice([1, 2, 4, 8])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "sample":
        vocab = _log_int(rng, 500, 152000)
        case.update(dtype=rng.choice(["fp16", "bf16", "fp32"]), vocab=vocab, rows=_log_int(rng, 1, 30_000_000 // vocab)
                    if vocab > 30000 else _log_int(rng, 1, 1000), temperature=rng.uniform(0.3, 1.5),
                    top_k=rng.choice([0, 0, 1, _log_int(rng, 2, 400)]), top_p=rng.choice([1.0, 1.0, rng.uniform(0.3, 0.99)]),
                    min_p=rng.choice([0.0, 0.0, rng.uniform(0.001, 0.3)]))
        return case
    if op == "cache8":
        batch = _log_int(rng, 1, 128)
        top = _log_int(rng, 1, max(2, 16384 // batch))
        case.update(dtype=dtype, cache=rng.choice(["int8", "e4m3"]), hq=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv,
                    batch=batch, new_lo=max(1, top // 6), new_hi=top, past_lo=0, past_hi=_log_int(rng, 1, 2000))
        return case
    if op == "tree":
        top = _log_int(rng, 2, 250)
        case.update(batch=_log_int(rng, 1, 256), new_lo=max(1, top // 4), new_hi=top, spread=_log_int(rng, 1, 64),
                    window=rng.choice([0, 0, _log_int(rng, 1, 30)]))
        return case
    if op == "accept":
        layers = rng.choice([1, 2, 16, 28])
        case.update(dtype=dtype, hkv=hkv, layers=layers, batch=_log_int(rng, 1, min(128, 10000 // (layers * hkv))),
                    new_lo=5, new_hi=_log_int(rng, 6, 64), past_lo=1, past_hi=_log_int(rng, 2, 250),
                    spread=_log_int(rng, 1, 30))
        return case
    tree = rng.random() < 0.6
    batch, past = _log_int(rng, 1, 64), _log_int(rng, 64, 40000)
    new = _log_int(rng, 2, 120) if tree else rng.choice([1, 1, _log_int(rng, 1, 2000)])
    hq = hkv * rng.choice([1, 2, 3, 4, 8])
    # no dearer than the largest listed case, and the scores of one KV head within 4 GB
    most = min(500_000_000 // hq, 1_000_000_000 // (hq // hkv))
    while batch > 1 and (batch * (past + new) > 250000 or batch * new * (past + new) > most):
        batch = batch // 2
    while new > 1 and batch * new * (past + new) > most:
        new = new // 2
    case.update(dtype=dtype, cache=rng.choice(["int8", "e4m3", "16bit"]), hq=hq, hkv=hkv, batch=batch,
                new_lo=max(1, new // 4), new_hi=new, past_lo=max(1, past // 8), past_hi=past,
                spread=_log_int(rng, 1, 30) if tree else 0, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                window=_log_int(rng, 16, past) if rng.random() < 0.25 else 0)
    return case


# ------------------------------------------------------------------------------- sizes, trees
def _sizes(case):
    """New and cached (with the new) tokens of every sequence; they belong to the case, not to the seed."""
    rng = random.Random(case["lens"])
    new = [_log_int(rng, case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    ctx = [rng.randint(case.get("past_lo", 0), case.get("past_hi", 0)) + n for n in new]
    return np.array(new, np.int64), np.array(ctx, np.int64)


def _parents(case):
    """Each sequence's parents: a node's parent is one of the `spread` nodes before it."""
    rng = np.random.default_rng(case["lens"])
    new, _ = _sizes(case)
    out = []
    for n in new:
        i = np.arange(n)
        back = np.floor(rng.random(n) * np.minimum(i, case["spread"])).astype(np.int64) + 1
        out.append(np.where(i > 0, i - back, -1))
    return out


def _depths(case):
    out = []
    for par in _parents(case):
        depth = np.zeros(len(par), np.int64)
        for i in range(1, len(par)):
            depth[i] = depth[par[i]] + 1
        out.append(depth)
    return out


def _accepted(case):
    """Each sequence's accepted nodes behind the root. They lie behind the slots that their K and V
    move to, so that a second pass over the same pages finds them as the first did."""
    rng = np.random.default_rng(case["lens"] + 1)
    out = []
    for n in _sizes(case)[0]:
        length = int(rng.integers(0, min((n - 1) // 2, 12) + 1))
        out.append(np.sort(rng.choice(np.arange(length + 1, n), length, replace=False)))
    return out


def _visible(case):
    """(pairs of a token and a key that it sees, keys that any token of their sequence sees)"""
    new, ctx = _sizes(case)
    depths = _depths(case) if case["spread"] else [np.arange(n) for n in new]
    pairs = keys = 0
    for n, c, depth in zip(new, ctx, depths):
        past, w = c - n, case["window"] or 1 << 40
        first = np.maximum(past + depth - w + 1, 0)
        pairs += int(np.sum(np.maximum(past - first, 0) + np.minimum(depth + 1, w)))
        keys += int(c - min(int(first.min()), past))
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "sample":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * 24, "flops": 2 * values}
    new, ctx = _sizes(case)
    tokens = int(new.sum())
    if op == "tree":
        words = (int(new.max()) + 31) // 32
        return {"bytes": tokens * (4 + 4 + 4 * words), "flops": int(sum(d.sum() for d in _depths(case)))}
    hkv = case["hkv"]
    if op == "accept":
        moved = sum(len(a) for a in _accepted(case))
        return {"bytes": moved * case["layers"] * hkv * D * 2 * 2 * 2 + tokens * 4 * 4, "flops": tokens}
    hq = case["hq"]
    if op == "cache8":
        row, codes = (hq + 2 * hkv) * D * 2, 2 * hkv * (D + 4)
        return {"bytes": tokens * (row + hq * D * 2 + 2 * codes + 2 * hkv * D * 2 + 4), "flops": tokens * (hq + 3 * hkv) * D * 3}
    pairs, keys = _visible(case)
    per_key = 2 * D * 2 if case["cache"] == "16bit" else 2 * (D + 4)
    return {"bytes": tokens * hq * (2 * D * 2 + 4) + keys * hkv * per_key, "flops": 4 * D * hq * pairs}


# ------------------------------------------------------------------------------------- inputs
def _dtype(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]


def _int32(a):
    return torch.from_numpy(np.asarray(a).astype(np.int32)).cuda()


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


def _scales_of(x, kind):
    """Scale of every row of 128 values, and their codes."""
    top = x.float().abs().amax(-1)
    code = x.float() * Q[kind] / torch.where(top > 0, top, 1.0)[..., None]
    return top / Q[kind], (code.round() if kind == "int8" else code).to(CODES[kind])


def _masks(case):
    """Ancestor bits [tokens, words] int32 (bit j of row i: node i sees node j) and depths, as a server keeps them for a step."""
    new, _ = _sizes(case)
    words = (int(new.max()) + 31) // 32
    rows, depths = [], _depths(case)
    for par, depth in zip(_parents(case), depths):
        see = np.zeros((len(par), words * 32), bool)
        for i in range(len(par)):
            if par[i] >= 0:
                see[i] = see[par[i]]
            see[i, i] = True
        if case["window"]:
            behind = depth[:, None] - np.pad(depth, (0, words * 32 - len(depth)))
            see &= behind < case["window"]
        rows.append(np.packbits(see, axis=1, bitorder="little").view(np.uint32))
    return torch.from_numpy(np.concatenate(rows).view(np.int32)).cuda(), _int32(np.concatenate(depths))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, st = (_dtype(case) if "dtype" in case else None), {"case": case}

    def normal(*shape, dtype=None):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype or dt)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a broad bulk and, in every row, some words that the context asks for
        x = 2.5 * normal(rows, vocab, dtype=torch.float32)
        x = x + (uniform(rows, vocab) < 12 / vocab) * (4.0 + 8.0 * uniform(rows, vocab))
        st["logits"] = x.to(dt)
        st["u"] = uniform(rows)
        # every request has settings of its own; some of them take the greatest logit
        st["temperature"] = torch.where(uniform(rows) < 0.1, 0.0, case["temperature"] * (0.7 + 0.6 * uniform(rows)))
        st["top_k"] = torch.where(uniform(rows) < 0.8, case["top_k"], 0).to(torch.int32)
        st["top_p"] = torch.where(uniform(rows) < 0.8, case["top_p"], 1.0)
        st["min_p"] = torch.where(uniform(rows) < 0.8, case["min_p"], 0.0)
        return st
    new, ctx = _sizes(case)
    tokens = int(new.sum())
    st["cu"], st["ctx"] = _int32(np.concatenate([[0], np.cumsum(new)])), _int32(ctx)
    if case["op"] == "tree":
        # as _parents() has them, but from the seed; a few nodes are roots as well, that is other first tokens
        node = _int32(np.concatenate([np.arange(n) for n in new]))
        back = (uniform(tokens) * node.clamp(max=case["spread"])).floor().int() + 1
        st["parents"] = torch.where((node == 0) | (uniform(tokens) < 0.02), -1, node - back)
        return st
    hkv = case["hkv"]
    st["table"], pool = _tables(g, ctx)
    if case["op"] == "accept":
        parents, sampled = _parents(case), []
        order = torch.stack([torch.randperm(4096, generator=g, device="cuda") for _ in new])
        tokens_of = order[:, :int(new.max())].cpu().numpy()
        for b, (n, path) in enumerate(zip(new, _accepted(case))):
            own_path = np.concatenate([[0], path]).astype(np.int64)
            parents[b][own_path[1:]] = own_path[:-1]
            follow = np.full(n, 5000)
            follow[own_path[:-1]] = tokens_of[b, own_path[1:]]
            sampled.append(follow)
        st["tokens"] = _int32(np.concatenate([tokens_of[b, :n] for b, n in enumerate(new)]))
        st["parents"], st["sampled"] = _int32(np.concatenate(parents)), _int32(np.concatenate(sampled))
        st["k"], st["v"] = normal(case["layers"], pool, PAGE, hkv, D), normal(case["layers"], pool, PAGE, hkv, D)
        return st
    hq = case["hq"]
    if case["op"] == "cache8":
        st["qkv"] = normal(tokens, hq + 2 * hkv, D)
        st["qkv"] = (st["qkv"] * torch.exp(normal(tokens, hq + 2 * hkv, 1).float()).to(dt)).view(tokens, -1)
        rows = 20000
        freq = 1.0 / (500000.0 ** (torch.arange(0, D, 2, device="cuda").double() / D))
        angle = torch.outer(torch.arange(rows, device="cuda").double(), freq)
        angle = torch.cat([angle, angle], dim=-1)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        st["positions"] = torch.randint(0, rows, (1, tokens), generator=g, device="cuda", dtype=torch.int32)
        for x in "kv":
            st[x + "_cache"] = torch.zeros(pool, PAGE, hkv, D, dtype=CODES[case["cache"]], device="cuda")
            st[x + "_scale"] = torch.zeros(pool, hkv, PAGE, device="cuda")
        return st
    st["q"] = normal(tokens, hq, D)
    st["mask"], st["depths"] = _masks(case) if case["spread"] else (None, None)
    if case["window"] and not case["spread"]:
        st["depths"] = _int32(np.concatenate([np.arange(n) for n in new]))
    st["k_scale"] = st["v_scale"] = None
    for x in "kv":
        rows = normal(pool, PAGE, hkv, D)
        if case["cache"] != "16bit":
            # tokens differ in size, as they do after a projection
            rows = rows * torch.exp(0.3 * normal(pool, PAGE, hkv, 1).float()).to(dt)
            scale, rows = _scales_of(rows, case["cache"])
            st[x + "_scale"] = scale.transpose(1, 2).contiguous()
        st[x + "_cache"] = rows
    return st


# -------------------------------------------------------------------------------- plain forms
def _padded(st):
    """Row indexes of every sequence's new tokens, padded: index [B, N] into the packed rows, which are real."""
    new = (st["cu"][1:] - st["cu"][:-1]).long()
    i = torch.arange(int(_sizes(st["case"])[0].max()), device="cuda")
    real = i < new[:, None]
    return torch.where(real, st["cu"][:-1].long()[:, None] + i, 0), real


def _slots(st):
    """Page and place of every new token, packed."""
    index, real = _padded(st)
    new = (st["cu"][1:] - st["cu"][:-1]).long()
    slot = ((st["ctx"].long() - new)[:, None] + torch.arange(index.shape[1], device="cuda"))[real]
    b = torch.arange(len(new), device="cuda")[:, None].expand(index.shape)[real]
    return st["table"].long()[b, slot // PAGE], slot % PAGE


def _plain_cache8(st):
    case = st["case"]
    hq, hkv, dt = case["hq"], case["hkv"], st["qkv"].dtype
    x = st["qkv"].float().view(-1, hq + 2 * hkv, D)
    cos, sin = (st[t][st["positions"][0].long()][:, None] for t in ("cos", "sin"))
    rot = x[:, :hq + hkv]
    rot = rot * cos + torch.cat([-rot[..., D // 2:], rot[..., :D // 2]], dim=-1) * sin
    page, place = _slots(st)
    k_scale, k_codes = _scales_of(rot[:, hq:], case["cache"])
    v_scale, v_codes = _scales_of(x[:, hq + hkv:], case["cache"])
    st["k_cache"][page, place], st["v_cache"][page, place] = k_codes, v_codes
    st["k_scale"][page, :, place], st["v_scale"][page, :, place] = k_scale, v_scale
    k = st["k_cache"][page, place].float() * st["k_scale"][page, :, place][..., None]
    v = st["v_cache"][page, place].float() * st["v_scale"][page, :, place][..., None]
    return rot[:, :hq].to(dt), k.to(dt), v.to(dt)


def _plain_tree(st):
    case = st["case"]
    index, real = _padded(st)
    n = index.shape[1]
    node = torch.arange(n, device="cuda")
    parent = st["parents"].long()[index]
    # steps of 0 or 1 to a node's parent, doubled until they reach every ancestor
    reach = ((parent[..., None] == node) | (node[:, None] == node)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    depth = reach.sum(-1) - 1
    if case["window"]:
        reach = reach * (depth[..., None] - depth[:, None] < case["window"])
    words = (n + 31) // 32
    bits = torch.nn.functional.pad(reach, (0, words * 32 - n)).long().view(*reach.shape[:2], words, 32)
    bits = (bits << torch.arange(32, device="cuda")).sum(-1)
    bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits)
    return bits[real].to(torch.int32), depth[real].to(torch.int32)


def _head_chunks(st):
    """KV heads in runs whose scores stay within 2 GB."""
    case = st["case"]
    each = case["batch"] * int(_sizes(case)[0].max()) * (case["hq"] // case["hkv"]) * st["table"].shape[1] * PAGE
    step = max(1, min(case["hkv"], (1 << 29) // each))
    return [slice(h, min(h + step, case["hkv"])) for h in range(0, case["hkv"], step)]


def _rows_of(st, x, heads):
    """Cached rows [B, h, C, D] of a run of heads, in 32 bits."""
    pages = st["table"].clamp(min=0).long()
    rows = st[x + "_cache"][pages, :, heads].float()  # [B, pages, 64, h, D]
    if st[x + "_scale"] is not None:
        rows = rows * st[x + "_scale"][pages, heads].transpose(2, 3)[..., None]
    b, p, _, h, _ = rows.shape
    return rows.permute(0, 3, 1, 2, 4).reshape(b, h, p * PAGE, D)


def _seen(st, index, real):
    """[B, N, C]: which cached tokens each new one sees."""
    case = st["case"]
    new = (st["cu"][1:] - st["cu"][:-1]).long()[:, None, None]
    past = st["ctx"].long()[:, None, None] - new
    i = torch.arange(index.shape[1], device="cuda")[:, None]
    j = torch.arange(st["table"].shape[1] * PAGE, device="cuda")
    node = (j - past).clamp(min=0, max=index.shape[1] - 1).expand(index.shape[0], index.shape[1], -1)
    if st["mask"] is None:
        see, depth = node <= i, i
        if case["window"]:
            see = see & (i - node < case["window"])
    else:
        words = st["mask"][index].long().gather(2, node // 32)
        see, depth = ((words >> (node % 32)) & 1).bool(), st["depths"].long()[index][..., None]
    before = j < past
    if case["window"]:
        before = before & (j > past + depth - case["window"])
    return torch.where(j < past, before, see & (j < past + new)) & real[..., None]


def _plain_attend(st):
    case = st["case"]
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    index, real = _padded(st)
    b, n = index.shape
    see = _seen(st, index, real)[:, None, :, None]
    o = torch.empty(b, n, hkv, group, D, device="cuda")
    lse = torch.empty(b, n, hkv, group, device="cuda")
    for heads in _head_chunks(st):
        q = st["q"].view(-1, hkv, group, D)[index][:, :, heads].float().permute(0, 2, 1, 3, 4)
        h = q.shape[1]
        s = torch.matmul(q.reshape(b, h, n * group, D), _rows_of(st, "k", heads).transpose(2, 3)) * D ** -0.5
        if case["softcap"]:
            s = case["softcap"] * torch.tanh(s / case["softcap"])
        s = s.view(b, h, n, group, -1).masked_fill(~see, -math.inf).view(b, h, n * group, -1)
        top = s.amax(-1, keepdim=True)
        top = torch.where(top > -math.inf, top, 0.0)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        out = torch.matmul(e, _rows_of(st, "v", heads)) / torch.where(total > 0, total, 1.0)
        o[:, :, heads] = out.view(b, h, n, group, D).permute(0, 2, 1, 3, 4)
        lse[:, :, heads] = (top + torch.log(total)).view(b, h, n, group).permute(0, 2, 1, 3)
    return o[real].view(-1, case["hq"], D).to(st["q"].dtype), lse[real].view(-1, case["hq"])


def _plain_sample(st):
    x = st["logits"].double()
    rows, vocab = x.shape
    greedy = (st["temperature"] == 0)[:, None]
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = order.values[:, :1]
    t = torch.where(greedy, 1.0, st["temperature"].double()[:, None])
    rank = torch.arange(vocab, device="cuda")
    k = torch.where(st["top_k"] > 0, st["top_k"], vocab).long()[:, None]
    w = torch.exp((order.values - top) / t)
    kept = rank < torch.where(greedy, 1, k)
    mass = (w * kept).cumsum(-1)
    kept = kept & (mass - w < st["top_p"].double()[:, None] * mass[:, -1:]) & (w >= st["min_p"].double()[:, None])
    kept[:, 0] = True
    live = torch.empty_like(kept).scatter_(1, order.indices, kept)
    run_mass = (torch.exp((x - top) / t) * live).cumsum(-1)
    hit = live & (run_mass > st["u"].double()[:, None] * run_mass[:, -1:])
    return hit.int().argmax(-1).to(torch.int32)


def _plain_accept(st):
    case = st["case"]
    index, real = _padded(st)
    b, n = index.shape
    parent = torch.where(real, st["parents"].long()[index], -1)
    token, want = st["tokens"][index], st["sampled"][index]
    node = torch.arange(n, device="cuda")
    # a node is accepted when it is the root, or its parent is and its token is the one sampled there;
    # of equal siblings the first
    good = (parent >= 0) & (token == want.gather(1, parent.clamp(min=0)))
    twin = good[:, :, None] & good[:, None] & (parent[:, :, None] == parent[:, None]) & (node < node[:, None])
    good = good & ~twin.any(-1)
    step = torch.where(good, parent, node)  # to the parent while that holds, else to itself
    for _ in range(max(1, (n - 1).bit_length())):
        step = step.gather(1, step)
    taken = (step == 0) & real
    counts = taken.sum(1)
    path = torch.sort(torch.where(taken, node, n), dim=1).values
    last = path.gather(1, (counts - 1)[:, None])
    follow = want.gather(1, last)[:, 0]
    live = path < n
    past = st["ctx"].long() - (st["cu"][1:] - st["cu"][:-1]).long()
    src = past[:, None] + torch.where(live, path, 0)
    dst = past[:, None] + node
    which = torch.arange(b, device="cuda")[:, None].expand(b, n)[live]
    src, dst = src[live], dst[live]
    table = st["table"].long()
    for x in "kv":
        st[x][:, table[which, dst // PAGE], dst % PAGE] = st[x][:, table[which, src // PAGE], src % PAGE]
    return torch.where(live, path, -1)[real].to(torch.int32), counts.to(torch.int32), follow, st["k"], st["v"]


def run(state):
    st, case = state, state["case"]
    if own:
        return _own(st, case)
    if case["op"] == "cache8":
        return _plain_cache8(st)
    if case["op"] == "tree":
        return _plain_tree(st)
    if case["op"] == "attend":
        return _plain_attend(st)
    if case["op"] == "sample":
        return _plain_sample(st)
    return _plain_accept(st)


def _own(st, case):
    if case["op"] == "cache8":
        from fast_infer_b200.kernels.rope import read_kv, rope_axes_store
        q = rope_axes_store(st["qkv"], case["hq"], st["cos"], st["sin"], st["positions"], (64,), st["k_cache"],
                            st["v_cache"], st["table"], PAGE, st["cu"], st["ctx"], k_scale=st["k_scale"],
                            v_scale=st["v_scale"])
        return (q, *read_kv(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"], st["table"], PAGE, st["cu"],
                            st["ctx"], st["qkv"].shape[0], dtype=st["qkv"].dtype))
    if case["op"] == "tree":
        from fast_infer_b200.kernels.drafting import draft_tree
        return draft_tree(st["parents"], st["cu"], int(_sizes(case)[0].max()), window=case["window"])
    if case["op"] == "attend":
        from fast_infer_b200.kernels.attention import paged_tree_attention
        return paged_tree_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], PAGE, st["cu"], st["ctx"],
                                    tree_mask=st["mask"], depths=st["depths"] if case["window"] else None,
                                    k_scale=st["k_scale"], v_scale=st["v_scale"], softcap=case["softcap"],
                                    window=case["window"], return_lse=True)
    if case["op"] == "sample":
        from fast_infer_b200.kernels.sampling import sample_tokens
        return sample_tokens(st["logits"], st["u"], st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                             min_p=st["min_p"])
    from fast_infer_b200.kernels.drafting import accept_drafts, keep_accepted
    path, counts, follow = accept_drafts(st["tokens"], st["sampled"], st["parents"], st["cu"])
    keep_accepted(st["k"], st["v"], st["table"], PAGE, st["cu"], st["ctx"], path, counts)
    return path, counts, follow, st["k"], st["v"]


# ------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "cache8":
        return _exact_cache8(st, case)
    if case["op"] == "attend":
        return _exact_attend(st, case)
    if case["op"] == "sample":
        return _exact_sample(st, case)
    if case["op"] == "accept":
        return _exact_accept(st, case)
    masks, depths = [], []
    cu, parents = st["cu"].tolist(), st["parents"].tolist()
    words = (int(_sizes(case)[0].max()) + 31) // 32
    for lo, hi in zip(cu, cu[1:]):
        for i in range(hi - lo):
            chain = [i]
            while parents[lo + chain[-1]] >= 0:
                chain.append(parents[lo + chain[-1]])
            depths.append(len(chain) - 1)
            bits = sum(1 << j for j in chain[:case["window"] or len(chain)])
            masks.append([(bits >> (32 * w)) & 0xffffffff for w in range(words)])
    masks = torch.tensor(masks, dtype=torch.int64, device="cuda")
    return torch.where(masks >= 2 ** 31, masks - 2 ** 32, masks).to(torch.int32), _int32(depths)


def _exact_cache8(st, case):
    hq, hkv, half = case["hq"], case["hkv"], D // 2
    x = st["qkv"].double().view(-1, hq + 2 * hkv, D)
    at = st["positions"][0].long()
    cos, sin = st["cos"].double()[at][:, None], st["sin"].double()[at][:, None]
    lo, hi = x[..., :half], x[..., half:]
    rot = torch.cat([lo * cos[..., :half] - hi * sin[..., :half], hi * cos[..., half:] + lo * sin[..., half:]], -1)

    def held(rows):
        top = rows.abs().amax(-1, keepdim=True)
        z = rows / torch.where(top > 0, top, 1.0) * Q[case["cache"]]
        if case["cache"] == "int8":
            step = torch.ones_like(z)
        else:  # three bits behind the leading one, 2^-9 the smallest step
            step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(z / step) * step * (top / Q[case["cache"]])
    return rot[:, :hq], held(rot[:, hq:hq + hkv]), held(x[:, hq + hkv:])


def _exact_attend(st, case):
    new, ctx = _sizes(case)
    if int(new.sum()) * int(ctx.max()) * case["hq"] > 20_000_000_000:
        return None
    hq, hkv = case["hq"], case["hkv"]
    trees = _parents(case) if case["spread"] else [np.arange(n) - 1 for n in new]
    o = torch.zeros(int(new.sum()), hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(int(new.sum()), hq, dtype=torch.float64, device="cuda")
    start = 0
    for b, (n, c, par) in enumerate(zip(new.tolist(), ctx.tolist(), trees)):
        window = case["window"] or 1 << 40
        hidden = np.ones((n, c), bool)
        for i in range(n):
            node, left = i, window
            while node >= 0 and left > 0:
                hidden[i, c - n + node] = False
                node, left = par[node], left - 1
            if left > 0:
                hidden[i, max(0, c - n - left):c - n] = False
        hidden = torch.from_numpy(hidden).cuda()
        pages = st["table"][b, :(c + PAGE - 1) // PAGE].long()
        rows = slice(start, start + n)
        for h in range(hkv):
            kv = []
            for x in "kv":
                y = st[x + "_cache"][pages][:, :, h].to(torch.float64).reshape(-1, D)
                if case["cache"] != "16bit":
                    y = y * st[x + "_scale"][pages, h].double().reshape(-1, 1)
                kv.append(y[:c])
            for head in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                s = st["q"][rows, head].double() @ kv[0].t() / math.sqrt(D)
                if case["softcap"]:
                    s = torch.tanh(s / case["softcap"]) * case["softcap"]
                s[hidden] = -math.inf
                lse[rows, head] = torch.logsumexp(s, -1)
                o[rows, head] = torch.softmax(s, -1) @ kv[1]
        start += n
    return o, lse


def _exact_sample(st, case):
    x = st["logits"].double().cpu().numpy()
    u, t, p, m = (st[n].double().cpu().numpy() for n in ("u", "temperature", "top_p", "min_p"))
    out = np.zeros(len(x), np.int32)
    for r, row in enumerate(x):
        if t[r] == 0:
            out[r] = np.argmax(row)
            continue
        k = int(st["top_k"][r]) or len(row)
        w = np.exp((row - row.max()) / t[r])
        order = np.argsort(-row, kind="stable")[:k]
        before = np.concatenate([[0.0], np.cumsum(w[order])])
        keep = order[(before[:-1] < p[r] * before[-1]) & (w[order] >= m[r])]
        keep = np.sort(keep if len(keep) else order[:1])
        total = np.cumsum(w[keep])
        out[r] = keep[min(int(np.searchsorted(total, u[r] * total[-1], side="right")), len(keep) - 1)]
    return torch.from_numpy(out).cuda()


def _exact_accept(st, case):
    cu, ctx = st["cu"].tolist(), st["ctx"].tolist()
    tokens, sampled, parents = st["tokens"].tolist(), st["sampled"].tolist(), st["parents"].tolist()
    path, counts, follow = [-1] * cu[-1], [], []
    k, v, table = st["k"], st["v"], st["table"].tolist()
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        nodes = [0]
        while True:
            want = sampled[lo + nodes[-1]]
            child = [i for i in range(hi - lo) if parents[lo + i] == nodes[-1] and tokens[lo + i] == want]
            if not child:
                break
            nodes.append(child[0])
        past = ctx[b] - (hi - lo)
        for d, node in enumerate(nodes):
            path[lo + d] = node
            to, at = past + d, past + node
            for x in (k, v):
                x[:, table[b][to // PAGE], to % PAGE] = x[:, table[b][at // PAGE], at % PAGE]
        counts.append(len(nodes))
        follow.append(sampled[lo + nodes[-1]])
    return _int32(path), _int32(counts), _int32(follow), k, v
