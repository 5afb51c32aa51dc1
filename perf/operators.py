"""The operators of the cache in 8 bits, as a server calls them: appending a step's keys and values (per-head norm and rotation on the
way), attention of single queries over the cache, and attention of prompts' portions over it.

The cache holds e4m3 numbers in blocks of 16 tokens: for every block and kv head one scale for the keys and one for the values, the
power of two 2^e with the smallest e in -100..119 for which the largest magnitude is at most 448 * 2^e.  A call that fills a block from its first
place starts it anew; one that goes on in a block lets its scale grow, and what the block held is rounded to the new scale.

    k_pages  [pages, KV, page, D]          v_pages  [pages, KV, page / 16, D, 16]          scales  fp32 [pages, KV, page / 16]

A case says how many requests bring one token (`singles`, with `low` to `high` tokens of context, their own included) and how many bring a portion
of a prompt (`portions` of `few` to `many` tokens behind `near` to `far` cached ones); lengths are drawn from the case alone.  Sizes of heads are
those of the benchmark's Qwen3 models and of the tests."""

import json
import math
import random

import numpy as np
import torch

own = False

E4M3, BF16, F32, F64, I32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.float64, torch.int32
DEV = "cuda:0"
BLOCK, TILE = 16, 64  # tokens that share a scale; queries of one work item of a portion
LEAST, MOST = -100, 119  # of a scale's exponent
EPS, THETA = 1e-6, 1e6


def _case(name=None, op="single", heads=32, kv_heads=8, dim=128, rotary=None, norm=True, page=16, singles=0, low=0, high=0,
          portions=0, few=0, many=0, near=0, far=0, window=0, cap=0.0, sink=False):  # fmt: skip
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, rotary=dim if rotary is None else rotary, norm=norm, page=page, singles=singles,
                low=low, high=high, portions=portions, few=few, many=many, near=near, far=far, window=window, cap=cap, sink=sink)  # fmt: skip
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # a token of one user's chat goes into the cache: nothing but latency
        _case("append-1", "append", 16, 8, singles=1, low=101, high=101),
        # a loaded server's decode step: 64 requests, each somewhere within a block
        _case("append-64", "append", singles=64, low=17, high=512),
        # the headline prompt, into empty pages
        _case("append-prompt-2048", "append", portions=1, few=2048, many=2048),
        # a step of everything: ragged portions that begin within a block beside single tokens; heads turned by half, without norms
        _case("append-ragged", "append", 40, 8, rotary=64, norm=False, page=32, singles=21, low=5, high=300, portions=5, few=33, many=700,
              near=3, far=250),  # fmt: skip
        # one user's chat with the smallest model
        _case("single-1-700", "single", 16, 8, singles=1, low=700, high=700),
        # the headline point, at odd lengths
        _case("single-8-2k", "single", singles=8, low=1500, high=2048),
        # a loaded server: requests at every stage of their lives; this is what the cache's bytes are for
        _case("single-64-ragged", "single", singles=64, low=300, high=8000),
        # one long document, cut along its keys over the whole GPU
        _case("single-1-131k", "single", 64, 8, singles=1, low=131005, high=131005),
        # narrow heads in groups of seven behind a window, capped scores, a sink, larger pages
        _case("single-narrow", "single", 28, 4, 64, page=64, singles=37, low=40, high=6000, window=2048, cap=30.0, sink=True),
        # a short question: time to the first token
        _case("prompt-333", "prompt", 16, 8, portions=1, few=333, many=333),
        # several users' portions meet in one step, behind prefixes of their own
        _case("prompt-ragged", "prompt", 32, 8, portions=6, few=40, many=600, near=0, far=5000),
        # the last portion of a long document
        _case("prompt-2048-behind-14k", "prompt", 32, 8, portions=1, few=2048, many=2048, near=14336, far=14336),
    ]


HEADS = ((16, 8, 128), (32, 8, 128), (40, 8, 128), (64, 8, 128), (8, 8, 128), (16, 4, 64), (28, 4, 64), (8, 1, 64), (24, 8, 192), (8, 4, 256))


def _spread(rng, low, high):
    """A whole number between low and high, evenly over its logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("append", "single", "prompt"))
    heads, kv_heads, dim = rng.choice(HEADS)
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 16, 32, 64)))
    if op == "append":
        case.update(rotary=rng.choice((dim, dim, dim // 2)), norm=rng.random() < 0.7)
        kind = rng.choice(("singles", "portions", "both"))
        if kind != "portions":
            case.update(singles=_spread(rng, 1, 256), low=1, high=_spread(rng, 2, 500))
        if kind != "singles":
            case.update(portions=rng.randint(1, 4), few=2, many=_spread(rng, 9, 500), near=0, far=rng.choice((0, 100)))
        return _case(**case)
    case.update(window=rng.choice((0, 0, 0, _spread(rng, 20, 4000))), cap=rng.choice((0.0, 0.0, 20.0)), sink=rng.random() < 0.25)
    if op == "single":
        singles = _spread(rng, 1, 128)
        high = _spread(rng, 2, min(60000, 400000 // singles))
        case.update(singles=singles, low=max(1, high // rng.choice((1, 3, 20))), high=high)
    else:
        portions = rng.randint(1, 6)
        many = _spread(rng, 9, 2000 // portions)
        case.update(portions=portions, few=max(1, many // rng.choice((1, 4))), many=many, near=0, far=rng.choice((0, _spread(rng, 10, 8000))))
    return _case(**case)


def _rows(case):
    """(tokens, tokens in the cache before them) of every request: portions first, then single tokens."""
    rng = random.Random(json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True))
    rows = [(rng.randint(case["few"], case["many"]), rng.randint(case["near"], case["far"])) for _ in range(case["portions"])]
    return rows + [(1, rng.randint(case["low"], case["high"]) - 1) for _ in range(case["singles"])]


def _seen(case, rows):
    """Keys that all queries see, and keys that a request's queries see together, added up over the requests."""
    pairs = union = 0
    for n, start in rows:
        at = np.arange(start, start + n)
        first = np.maximum(0, at - case["window"] + 1) if case["window"] else np.zeros(n, dtype=np.int64)
        pairs += int((at + 1 - first).sum())
        union += int(start + n - first[0])
    return pairs, union


def work(case):
    rows, (H, KV, D) = _rows(case), (case["heads"], case["kv_heads"], case["dim"])
    T = sum(n for n, _ in rows)
    if case["op"] == "append":  # the projection in, queries out, keys and values in 8 bits, angles
        return {"bytes": T * (2 * (H + 2 * KV) * D + 2 * H * D + 2 * KV * D + 4 * case["rotary"]), "flops": T * (H + KV) * D * 8}
    pairs, union = _seen(case, rows)
    return {"bytes": union * KV * D * 2 + 4 * T * H * D, "flops": 4 * H * D * pairs}


# ---- what a server has in hand ---------------------------------------------------------------------


def _scale_of(amax):
    """2^e, e the smallest in LEAST..MOST with amax <= 448 * 2^e."""
    half, e = torch.frexp(amax)  # amax = half * 2^e, half in [0.5, 1)
    e = torch.where(amax > 0, e - 9 + (half > 0.875).int(), LEAST).clamp(LEAST, MOST)
    return torch.ldexp(torch.ones_like(amax), e)


def _to_blocks(x):
    """Numbers [pages, KV, blocks, 16, D] as e4m3 and their blocks' scales."""
    scale = _scale_of(x.abs().amax((-1, -2)).float())
    return (x.float() / scale[..., None, None]).clamp(-448, 448).to(E4M3), scale


def _inv_freq(rotary):
    return THETA ** (-torch.arange(0, rotary, 2, dtype=F64, device=DEV) / rotary)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, bs = _rows(case), case["page"]
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    R, T = len(rows), sum(n for n, _ in rows)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    ends = [start + n for n, start in rows]
    width = -(-max(ends) // bs)
    need = [-(-e // bs) for e in ends]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).int().cpu()
    tables = torch.zeros(R, width, dtype=I32)
    at = 0
    for r, n in enumerate(need):
        tables[r, :n] = order[at : at + n]
        at += n
    row = torch.repeat_interleave(torch.arange(R), torch.tensor([n for n, _ in rows]))
    positions = torch.cat([torch.arange(start, start + n) for n, start in rows])
    tiles = [(at, min(TILE, n - q), r, start + q) for r, ((n, start), first) in enumerate(zip(rows, np.cumsum([0] + [n for n, _ in rows])))
             for q in range(0, n, TILE) for at in (int(first) + q,)]  # fmt: skip
    tiles.sort(key=lambda t: -(t[3] + t[1]))  # those that see most keys first, as the engine packs a step
    longest = torch.argsort(-positions, stable=True)
    # keys have a few coordinates that are larger than the others', values do not
    loud = 1 + 5 * (torch.rand(1, KV, 1, 1, D, generator=g, device=DEV) < 0.04)
    nb = bs // BLOCK
    k, k_scales = _to_blocks(randn(pages, KV, nb, BLOCK, D) * loud)
    v, v_scales = _to_blocks(randn(pages, KV, nb, BLOCK, D) * (0.2 + randn(pages, KV, nb, 1, 1).abs()))
    state = dict(case=case, k=k.view(pages, KV, bs, D), v=v.view(torch.uint8).transpose(-1, -2).contiguous().view(E4M3), ks=k_scales, vs=v_scales,
                 tables=tables.to(DEV), row=row.int().to(DEV), positions=positions.int().to(DEV), items=longest.int().to(DEV),
                 tiles=torch.tensor(tiles, dtype=I32).view(-1, 4).to(DEV), context=max(ends), keys=sum(t[3] + t[1] for t in tiles),
                 most=max(n for n, _ in rows))  # fmt: skip
    if case["op"] == "append":
        state["qkv"] = randn(T, H + 2 * KV, D).to(BF16)
        state["slots"] = (tables[row, positions // bs] * bs + positions % bs).int().to(DEV)
        angles = positions.to(DEV)[:, None].double() * _inv_freq(case["rotary"])
        state["cos_sin"] = torch.stack([angles.cos(), angles.sin()], -1).float()
        state["gains"] = [(1 + 0.2 * randn(D)).to(BF16) for _ in range(2)] if case["norm"] else [None, None]
        return state
    state["q"] = (randn(T, H, D) * 1.3).to(BF16)
    state["sink"] = randn(H) if case["sink"] else False
    state["scale"] = D**-0.5
    return state


# ---- the framework's calls ---------------------------------------------------------------------------


def _own_append(s):
    from atomserve_amd.kernels import ops

    c, qkv = s["case"], s["qkv"]
    q = torch.empty((qkv.shape[0], c["heads"], c["dim"]), dtype=BF16, device=qkv.device)
    ops.qk_norm_rope_store8(qkv, *s["gains"], s["cos_sin"], s["slots"], q, s["k"], s["v"], s["ks"], s["vs"], c["heads"], c["kv_heads"], EPS)
    return q


def _own_single(s):
    from atomserve_amd.kernels import ops

    c, q = s["case"], s["q"]
    out = torch.empty_like(q)
    ops.attn_single_query8(q, s["k"], s["v"], s["ks"], s["vs"], s["items"], s["positions"], None, s["tables"], out, s["scale"], c["window"],
                           s["context"], softcap=c["cap"], sink=s["sink"])  # fmt: skip
    return out


def _own_prompt(s):
    from atomserve_amd.kernels import ops

    c, q = s["case"], s["q"]
    out = torch.empty_like(q)
    ops.attn_prefill8(q, s["k"], s["v"], s["ks"], s["vs"], s["tiles"], s["tables"], out, s["scale"], c["window"], s["context"],
                      tile_keys=s["keys"], softcap=c["cap"], sink=s["sink"])  # fmt: skip
    return out


# ---- the same in elementary operations -----------------------------------------------------------------


def _plain_heads(x, gain, cos_sin):
    """Heads [T, N, D] in 32 bits, normed and turned."""
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.float()
    half = cos_sin.shape[1]
    a, b, rest = x[..., :half], x[..., half : 2 * half], x[..., 2 * half :]
    c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1)


def _plain_put(pages, scales, x, slots, bs, values):
    """x [T, KV, D] into the blocks that `slots` name; pages as bytes, in place."""
    KV, D, nb = x.shape[1], x.shape[2], bs // BLOCK
    x = torch.where(torch.isfinite(x), x, 0.0)
    page, sub, place = (slots // bs).long(), (slots % bs // BLOCK).long(), (slots % BLOCK).long()
    flat = page * nb + sub
    ids, which = torch.unique(flat, return_inverse=True)
    p, b = ids // nb, ids % nb
    amax = torch.zeros(ids.numel(), KV, device=x.device).index_reduce_(0, which, x.abs().amax(-1), "amax")
    new = torch.zeros(ids.numel(), device=x.device).index_reduce_(0, which, (place == 0).float(), "amax") > 0
    old = torch.where(new[:, None], 0.0, scales[p, :, b])
    scale = torch.maximum(old, _scale_of(amax))
    # what the blocks held, at their new scale
    if values:
        held = pages[p, :, b]
    else:
        held = pages.view(-1, KV, nb, BLOCK, D)[p, :, b]
    ratio = (old / scale)[:, :, None, None]
    kept = torch.where((ratio > 0) & (ratio < 1), (held.view(E4M3).float() * ratio).to(E4M3).view(torch.uint8), held)
    put = (x / scale[which][..., None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
    if values:
        pages[p, :, b] = kept
        pages[page, :, sub, :, place] = put
    else:
        pages.view(-1, KV, nb, BLOCK, D)[p, :, b] = kept
        pages[page, :, slots.long() % bs] = put
    scales[p, :, b] = scale


def _plain_append(s):
    c, x = s["case"], s["qkv"].float()
    H, KV = c["heads"], c["kv_heads"]
    q = _plain_heads(x[:, :H], s["gains"][0], s["cos_sin"])
    k = _plain_heads(x[:, H : H + KV], s["gains"][1], s["cos_sin"])
    _plain_put(s["k"].view(torch.uint8), s["ks"], k, s["slots"], c["page"], False)
    _plain_put(s["v"].view(torch.uint8), s["vs"], x[:, H + KV :], s["slots"], c["page"], True)
    return q.to(BF16)


def _gathered(s):
    """Keys and values [R, KV, L, D] of every request's pages, in 32 bits."""
    table = s["tables"].long()
    R, W = table.shape
    k, v, ks, vs = (s[name][table] if name in ("ks", "vs") else s[name].view(torch.uint8)[table].view(E4M3).float() for name in ("k", "v", "ks", "vs"))
    KV, bs, D = k.shape[2:]
    nb = bs // BLOCK
    k = k.view(R, W, KV, nb, BLOCK, D) * ks[..., None, None]
    v = v * vs[..., None, None]
    k = k.permute(0, 2, 1, 3, 4, 5).reshape(R, KV, W * bs, D)
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(R, KV, W * bs, D)
    return k, v


def _plain_attend(s):
    c, q = s["case"], s["q"].float()
    T, H, D = q.shape
    k, v = _gathered(s)
    R, KV, L, _ = k.shape
    row, N = s["row"].long(), s["most"]
    nth = torch.arange(T, device=q.device) - torch.searchsorted(row, row)  # a token's place in its row
    rows = torch.zeros(R, N, H, D, device=q.device)
    at = torch.zeros(R, N, dtype=torch.long, device=q.device)
    rows[row, nth] = q
    at[row, nth] = s["positions"].long()
    grouped = rows.view(R, N, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(R, KV, H // KV * N, D)
    scores = (torch.matmul(grouped, k.transpose(-1, -2).contiguous()) * s["scale"]).view(R, KV, H // KV, N, L)
    if c["cap"] > 0:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    key = torch.arange(L, device=q.device)
    seen = key <= at[..., None]
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    sink = s["sink"].view(1, KV, H // KV, 1, 1) if c["sink"] else None
    if sink is not None:
        top = torch.maximum(top, sink)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(weights.view(R, KV, H // KV * N, L), v).view(R, KV, H // KV, N, D) / total
    return out.permute(0, 3, 1, 2, 4).reshape(R, N, H, D)[row, nth].to(BF16)


def run(state):
    op = state["case"]["op"]
    if op == "append":
        q = _own_append(state) if own else _plain_append(state)
        return {"q": q, "k": state["k"], "v": state["v"], "k_scales": state["ks"], "v_scales": state["vs"]}
    if own:
        return _own_single(state) if op == "single" else _own_prompt(state)
    return _plain_attend(state)


# ---- the definition in 64 bits ---------------------------------------------------------------------------


def _exact_blocks(pages, scales, new):
    """Pages [..., 16 tokens, D] as numbers, and scales, after `new` ({(page, head-less block): {place: [KV, D]}}) has been put in."""
    for (page, block), places in new.items():
        amax = torch.stack([x.abs().amax(-1) for x in places.values()]).amax(0)
        e = torch.ceil(torch.log2(amax / 448)).clamp(LEAST, MOST)
        e = torch.where(amax > 448 * 2.0**e, e + 1, torch.where(amax <= 448 * 2.0 ** (e - 1), e - 1, e)).clamp(LEAST, MOST)
        scale = torch.where(amax > 0, 2.0**e, 2.0**LEAST)
        if 0 not in places:
            before = scales[page, :, block].clone()
            scale = torch.maximum(before, scale)
            pages[page, :, block] *= (before / scale)[:, None, None]
        for place, x in places.items():
            pages[page, :, block, place] = x / scale[:, None]
        scales[page, :, block] = scale


def exact(case, seed):
    s = prepare(case, seed)
    H, KV, D, bs = case["heads"], case["kv_heads"], case["dim"], case["page"]
    pages, nb = s["k"].shape[0], bs // BLOCK
    k = s["k"].double().view(pages, KV, nb, BLOCK, D)
    v = s["v"].double().transpose(-1, -2).contiguous()
    ks, vs = s["ks"].double(), s["vs"].double()
    if case["op"] == "append":
        x = s["qkv"].double()
        turn = s["cos_sin"].double()[:, None]
        half = case["rotary"] // 2
        heads = []
        for part, gain in ((x[:, :H], s["gains"][0]), (x[:, H : H + KV], s["gains"][1])):
            if gain is not None:
                part = part * gain.double() / part.square().mean(-1, keepdim=True).add(EPS).sqrt()
            first, second = part[..., :half].clone(), part[..., half : 2 * half].clone()
            part = part.clone()
            part[..., :half] = first * turn[..., 0] - second * turn[..., 1]
            part[..., half : 2 * half] = second * turn[..., 0] + first * turn[..., 1]
            heads.append(part)
        q, k_new, v_new = heads[0].cpu(), heads[1].cpu(), x[:, H + KV :].cpu()
        k, v, ks, vs = k.cpu(), v.cpu(), ks.cpu(), vs.cpu()
        puts = {}, {}
        for t, slot in enumerate(s["slots"].tolist()):
            at = (slot // bs, slot % bs // BLOCK)
            for put, new in zip(puts, (k_new, v_new)):
                put.setdefault(at, {})[slot % BLOCK] = new[t]
        _exact_blocks(k, ks, puts[0])
        _exact_blocks(v, vs, puts[1])
        return {"q": q, "k": k.view(pages, KV, bs, D), "v": v.transpose(-1, -2).contiguous(), "k_scales": ks, "v_scales": vs}
    k = (k * ks[..., None, None]).transpose(0, 1).reshape(KV, pages * bs, D)
    v = (v * vs[..., None, None]).transpose(0, 1).reshape(KV, pages * bs, D)
    q, out = s["q"].double(), torch.empty(s["q"].shape, dtype=F64, device=DEV)
    rows, first = _rows(case), 0
    for r, (n, start) in enumerate(rows):
        slots = (s["tables"][r].long()[:, None] * bs + torch.arange(bs, device=DEV)).view(-1)[: start + n]
        at = torch.arange(start, start + n, device=DEV)[:, None]
        key = torch.arange(start + n, device=DEV)[None]
        hidden = (key > at) | (key <= at - case["window"] if case["window"] else key < 0)
        for h in range(H):
            scores = q[first : first + n, h] @ k[h * KV // H, slots].T * D**-0.5
            if case["cap"]:
                scores = torch.tanh(scores / case["cap"]) * case["cap"]
            scores = scores.masked_fill(hidden, -math.inf)
            if case["sink"]:
                scores = torch.cat([scores, s["sink"][h].double().expand(n, 1)], 1)
            weights = torch.softmax(scores, 1)[:, : start + n]
            out[first : first + n, h] = weights @ v[h * KV // H, slots]
        first += n
    return out
