"""Operators of long texts in a bounded cache, as measurable cases.

A server whose requests outgrow their share of the paged cache runs, through
``pageserve_amd``:

``attend``   attention of a request's newest rows, one of a decoding step or
             thousands of a prompt's chunk, over the cached tokens of a sliding
             window and the first few, the cache in 16 bits or in 4
             (``window_attention``, ``window_attention4``).
``write``    key and value rows stored in 4 bits at their slots, and read back
             (``write_kv4``, ``read_kv4``).
``weigh``    what the rows' attention weights add up to for each cached token
             (``accumulate_weights``).
``evict``    requests cut to a budget of their tokens of largest weight, those
             moved together in every layer's cache (``evict_tokens``).

Sizes are those of the models this repository serves: 16 query and 2 key heads
of 128 ("3b"), 14 query and 2 key heads of 64 ("0.5b"), cache blocks of 16
tokens and more.

With ``own`` false the operators are computed in elementary torch operations,
in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import torch

own = False

#        query heads, key heads, head_dim
MODELS = {"3b": (16, 2, 128), "0.5b": (14, 2, 64)}
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
#: the values of the 4-bit codes 0..7 (code + 8 is the negative value)
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _attend_case(name, model, bits, requests, tokens, context, window, sinks, block, dtype, lse=False):
    return {"name": name, "kind": "attend", "model": model, "bits": bits, "requests": requests, "tokens": tokens,
            "context": context, "window": window, "sinks": sinks, "block": block, "dtype": dtype, "lse": lse}


def listed():
    return [
        # plain decoding of a few short chats with a small window
        _attend_case("attend-step-6", "0.5b", 16, 6, 1, 700, 256, 4, 16, "bf16"),
        # plain decoding of a full batch whose texts are longer than the window
        _attend_case("attend-step-48", "3b", 16, 48, 1, 12000, 4096, 4, 16, "bf16"),
        # chunks of four long prompts
        _attend_case("attend-prompt-4", "3b", 16, 4, 2048, 8000, 4096, 64, 64, "f16"),
        # one very long document in 4 bits, all of it visible
        _attend_case("attend4-step-1", "3b", 4, 1, 1, 120000, 0, 0, 16, "bf16"),
        # a full batch of long chats in 4 bits, weights to be accumulated
        _attend_case("attend4-step-32", "3b", 4, 32, 1, 16000, 0, 0, 32, "bf16", lse=True),
        # the next chunk of two documents in 4 bits
        _attend_case("attend4-prompt-2", "3b", 4, 2, 1024, 16000, 0, 0, 64, "bf16"),
        # one token of each request stored in 4 bits
        {"name": "write4-step-64", "kind": "write", "model": "0.5b", "rows": 64, "dtype": "bf16", "block": 16,
         "keep": 0.9},
        # a chunk of prompts stored in 4 bits, all rows
        {"name": "write4-prompts-8192", "kind": "write", "model": "3b", "rows": 8192, "dtype": "f16", "block": 64,
         "keep": 1.0},
        # weights of a decoding step
        {"name": "weigh-step-16", "kind": "weigh", "model": "3b", "bits": 16, "requests": 16, "tokens": 1,
         "context": 8000, "window": 0, "sinks": 0, "block": 16, "dtype": "bf16"},
        # weights of two chunks of prompts over a cache in 4 bits
        {"name": "weigh4-prompt-2", "kind": "weigh", "model": "3b", "bits": 4, "requests": 2, "tokens": 512,
         "context": 8192, "window": 0, "sinks": 0, "block": 64, "dtype": "bf16"},
        # one layer of four chats that have just passed their budget
        {"name": "evict-chats-4", "kind": "evict", "model": "0.5b", "bits": 16, "requests": 4, "context": 1100,
         "budget": 1024, "sinks": 4, "recent": 128, "layers": 1, "block": 16, "dtype": "bf16"},
        # long prompts cut to half, in the caches of several layers
        {"name": "evict-prompts-8", "kind": "evict", "model": "3b", "bits": 16, "requests": 8, "context": 8192,
         "budget": 4096, "sinks": 16, "recent": 512, "layers": 4, "block": 16, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "write", "weigh", "weigh", "evict"])
    case = {"kind": kind, "model": rng.choice(["3b", "3b", "0.5b"]), "block": rng.choice([16, 16, 32, 64, 128]),
            "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "write":
        return case | {"rows": _log_int(rng, 1, 8192), "keep": rng.choice([0.3, 0.9, 1.0])}
    case["bits"] = rng.choice([16, 4])
    if kind == "evict":
        requests, layers = _log_int(rng, 1, 32), rng.randint(1, 4)
        context = _log_int(rng, 64, min(60000, 260_000 // (requests * layers)))
        budget = max(1, int(context * rng.uniform(0.2, 1.0)))
        return case | {"requests": requests, "layers": layers, "context": context, "budget": budget,
                       "sinks": rng.choice([0, 4, rng.randint(0, budget)]),
                       "recent": rng.choice([0, budget // 8, rng.randint(0, budget)])}
    tokens = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 17, 2048)])
    requests = _log_int(rng, 1, min(48, max(1, 8192 // tokens)))
    # (as much as the largest listed cases at most)
    most = min(120000, (40 if kind == "attend" else 8) * 10**6 // (tokens * requests), 500_000 // requests)
    context = _log_int(rng, 1, max(most, tokens))
    case |= {"requests": requests, "tokens": tokens, "context": context,
             "window": rng.choice([0, _log_int(rng, 1, 8192)]), "sinks": rng.choice([0, 4, _log_int(rng, 1, 256)])}
    return case | {"lse": rng.random() < 0.5} if kind == "attend" else case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _even(lo, hi, n):
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _spread(gen, lo, hi, n):
    """n numbers spread evenly over lo..hi, in random order, int32"""
    return torch.tensor(_even(lo, hi, n), dtype=torch.int32, device="cuda")[
        torch.randperm(n, generator=gen, device="cuda")]


def _offsets(counts):
    """[0, c0, c0 + c1, ...] int32"""
    return torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)


def _tables(gen, lens, context, block):
    """Distinct random block ids for every request's tokens, -1 behind, and how many blocks there are."""
    blocks = (lens + block - 1) // block
    columns = (context + block - 1) // block
    pool = int(blocks.sum()) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    col = torch.arange(columns, device="cuda")
    at = (_offsets(blocks)[:-1, None] + col).clamp(max=pool - 1)
    return torch.where(col < blocks[:, None], order[at.long()], -1).to(torch.int32), pool


def _cache(gen, bits, pool, block, kv, dim, dt):
    """A layer's cache: keys and values, or the codes and scales of each as the 4-bit cache keeps them."""
    if bits == 16:
        return [_randn(gen, pool, block, kv, dim, dtype=dt) for _ in range(2)]
    parts = []
    for _ in range(2):
        # a row of 32 normal numbers has a largest one of about 2.2, a sixth of that is the scale
        scale = torch.rand((pool, kv, block, dim // 32), generator=gen, device="cuda") * 0.3 + 0.25
        parts += [torch.randint(0, 256, (pool, kv, block, dim // 2), generator=gen, device="cuda", dtype=torch.uint8),
                  _cut(scale).to(torch.bfloat16)]
    return parts


def _cut(x):
    """The first 6 significant bits of positive fp32 numbers."""
    return (x.view(torch.int32) & ~0x3FFFF).view(torch.float32)


def _attend_inputs(case, seed):
    gen, n, t, context = _gen(seed), case["requests"], case["tokens"], case["context"]
    heads, kv, dim = MODELS[case["model"]]
    dt = DTYPES[case["dtype"]]
    rows = _spread(gen, (t + 1) // 2, t, n)
    # (with its rows a request holds as many tokens at least)
    lens = torch.maximum(_spread(gen, (context + 1) // 2, context, n), rows)
    offsets = _offsets(rows)
    tables, pool = _tables(gen, lens, max(context, t), case["block"])
    state = {"q": _randn(gen, int(offsets[-1]), heads, dim, dtype=dt), "tables": tables, "lens": lens, "offsets": offsets,
             "cache": _cache(gen, case["bits"], pool, case["block"], kv, dim, dt), "new": rows, "dtype": dt,
             "tokens": t, "context": max(context, t), "window": case["window"], "sinks": case["sinks"],
             "bits": case["bits"], "block": case["block"]}
    if case["kind"] == "attend":
        state["lse"] = case["lse"]
    return state


def _weigh_inputs(case, seed):
    state = _attend_inputs(case, seed)
    state["lse"] = _scores(state)[0].logsumexp(-1)[_scores_live(state)]
    pool = state["cache"][0].shape[0]
    state["weights"] = torch.rand((pool, case["block"]), generator=_gen(seed + 1), device="cuda")
    return state


def _write_inputs(case, seed):
    gen, n, s = _gen(seed), case["rows"], case["block"]
    _, kv, dim = MODELS[case["model"]]
    dt = DTYPES[case["dtype"]]
    blocks = (n + s - 1) // s + 4
    slots = torch.randperm(blocks * s, generator=gen, device="cuda")[:n]
    if case["keep"] < 1:  # some rows have no slot: rejected drafts, requests that were not served
        slots = torch.where(torch.rand(n, generator=gen, device="cuda") < case["keep"], slots, -1)
    else:  # a prompt's rows fill whole blocks
        base = torch.randperm(blocks, generator=gen, device="cuda")
        at = torch.arange(n, device="cuda")
        slots = base[at // s] * s + at % s
    # (one block more than the slots reach)
    return {"k": _randn(gen, n, kv, dim, dtype=dt), "v": _randn(gen, n, kv, dim, dtype=dt), "slots": slots, "dtype": dt,
            "cache": _cache(gen, 4, blocks + 1, s, kv, dim, dt)}


def _evict_inputs(case, seed):
    gen, n, context = _gen(seed), case["requests"], case["context"]
    _, kv, dim = MODELS[case["model"]]
    lens = _spread(gen, (context * 3 + 3) // 4, context, n)
    tables, pool = _tables(gen, lens, context, case["block"])
    # a few tokens have most of the weight
    weights = torch.exp(2 * torch.randn((pool, case["block"]), generator=gen, device="cuda"))
    return {"lens": lens, "tables": tables, "weights": weights, "context": context, "sinks": case["sinks"],
            "recent": case["recent"], "budget": torch.full_like(lens, case["budget"]), "most": case["budget"],
            "slots": torch.arange(pool * case["block"], device="cuda"),
            "layers": [_cache(gen, case["bits"], pool, case["block"], kv, dim, DTYPES[case["dtype"]])
                       for _ in range(case["layers"])], "bits": case["bits"], "block": case["block"]}


_INPUTS = {"attend": _attend_inputs, "weigh": _weigh_inputs, "write": _write_inputs, "evict": _evict_inputs}


def prepare(case, seed):
    return _INPUTS[case["kind"]](case, seed) | {"kind": case["kind"]}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend, "weigh": _weigh, "write": _write, "evict": _evict}[state["kind"]](state)


def _run_own(s):
    import pageserve_amd as P

    kind = s["kind"]
    if kind == "write":
        cache = P.KVCache4.of(*s["cache"])
        P.write_kv4(s["k"], s["v"], cache, s["slots"])
        return P.read_kv4(cache, s["slots"], s["dtype"])
    if kind == "evict":
        weights = s["weights"].clone()
        layers = [[part.clone() for part in c] for c in s["layers"]]
        caches = [P.KVCache4.of(*c) if s["bits"] == 4 else tuple(c) for c in layers]
        kept = P.evict_tokens(weights, s["lens"], s["budget"], s["tables"], caches, sinks=s["sinks"],
                              recent=s["recent"], max_context=s["context"])
        # (of codes the values that they stand for)
        return kept, weights, [P.read_kv4(c, s["slots"]) for c in caches] if s["bits"] == 4 else layers
    cache = (P.KVCache4.of(*s["cache"]),) if s["bits"] == 4 else tuple(s["cache"])
    seen = {"window": s["window"] or None, "sinks": s["sinks"], "max_tokens": s["tokens"], "max_context": s["context"]}
    if kind == "weigh":
        weights = s["weights"].clone()
        P.accumulate_weights(s["q"], cache[0], s["tables"], s["lens"], s["offsets"], s["lse"], weights,
                             new_lens=s["new"], **seen)
        return weights
    attention = P.window_attention4 if s["bits"] == 4 else P.window_attention
    return attention(s["q"], *cache, s["tables"], s["lens"], s["offsets"], return_lse=s["lse"], **seen)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _nibbles(b):
    """uint8 [...] -> the codes' values fp32 [..., 2], the low half first"""
    value = torch.tensor(VALUES + tuple(-x for x in VALUES), device=b.device)
    return value[torch.stack((b & 15, b >> 4), -1).int()]


def _dense_k(codes, scale):
    """Keys of a 4-bit cache, fp32 [blocks, block_size, kv_heads, head_dim].  Byte 4 (dc a + c) + i of a row, dc = head_dim
    / 32, holds dims 32 c + 8 a + 2 i and the next one."""
    n, h, s, half = codes.shape
    dc = half // 16
    x = _nibbles(codes.reshape(n, h, s, 4, dc, 4)).permute(0, 2, 1, 4, 3, 5, 6).reshape(n, s, h, dc, 32)
    return (x * scale.permute(0, 2, 1, 3).float()[..., None]).flatten(3)


def _dense_v(codes, scale):
    """Values of a 4-bit cache.  Of 16 tokens, token 4 a + b has its dims i, 16 + i, 32 + i, ... together at
    ((16 a + i) 4 + b) head_dim / 32 bytes from the first."""
    n, h, s, half = codes.shape
    x = _nibbles(codes.view(n, h, s // 16, 4, 16, 4, half // 16)).permute(0, 2, 3, 5, 1, 6, 7, 4)
    x = x.reshape(n, s, h, half // 16, 32)
    return (x * scale.permute(0, 2, 1, 3).float()[..., None]).flatten(3)


def _gathered(s, dense):
    """Every request's cached tokens, padded to the longest: fp32 [requests, kv_heads, context, head_dim]"""
    pos = torch.arange(s["context"], device=dense.device)
    slot = s["tables"].long().clamp(min=0)[:, pos // s["block"]] * s["block"] + pos % s["block"]
    slot = slot * (pos < s["lens"][:, None])
    return dense.flatten(0, 1)[slot].float().permute(0, 2, 1, 3).contiguous()


def _rows(s):
    """(places of every request's rows, padded to the most; which of them are rows)"""
    rows = s["offsets"][:-1, None].long() + torch.arange(s["tokens"], device=s["q"].device)
    return rows.clamp(max=s["q"].shape[0] - 1), rows < s["offsets"][1:, None]


def _scores_live(s):
    return _rows(s)[1]


def _scores(s):
    """The scores of the padded rows, [requests, tokens, heads, context], -inf where a row does not see a token; and which
    it sees, [requests, tokens, context]."""
    rows, live = _rows(s)
    n, t = rows.shape
    heads, dim = s["q"].shape[1:]
    k = _gathered(s, _dense_k(*s["cache"][:2]) if s["bits"] == 4 else s["cache"][0])
    kv = k.shape[1]
    q = s["q"][rows].float().view(n, t, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * dim ** -0.5
    score = score.view(n, kv, t, heads // kv, -1).permute(0, 2, 1, 3, 4).reshape(n, t, heads, -1)
    at = (s["lens"] - s["new"])[:, None] + torch.arange(t, device=q.device)  # the rows' places in their texts
    pos = torch.arange(s["context"], device=q.device)
    sees = (pos <= at[..., None]) & live[..., None]
    if s["window"]:
        sees &= (pos > at[..., None] - s["window"]) | (pos < s["sinks"])
    return score.masked_fill_(~sees[:, :, None], float("-inf")), sees


def _attend(s):
    score, _ = _scores(s)
    n, t, heads, _ = score.shape
    v = _gathered(s, _dense_v(*s["cache"][2:]) if s["bits"] == 4 else s["cache"][1])
    kv, dim = v.shape[1], v.shape[3]
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    p = (p / total.clamp(min=1e-30)).view(n, t, kv, heads // kv, -1)
    p = p.permute(0, 2, 1, 3, 4).reshape(n, kv, t * heads // kv, -1)
    o = torch.matmul(p, v).view(n, kv, t, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(n, t, heads, dim)
    live = _scores_live(s)
    out = o[live].to(s["dtype"])
    return (out, (torch.log(total) + top).squeeze(-1)[live]) if s["lse"] else out


def _weigh(s):
    score, sees = _scores(s)
    rows, _ = _rows(s)
    p = torch.exp(score - s["lse"][rows][..., None])
    add = torch.where(sees[:, :, None], p, 0.0).sum((1, 2))  # [requests, context]
    pos = torch.arange(s["context"], device=add.device)
    inside = pos < s["lens"][:, None]
    slot = s["tables"].long()[:, pos // s["block"]] * s["block"] + pos % s["block"]
    # (a request's new tokens start from nothing)
    old = s["weights"].flatten()[slot.clamp(min=0)] * (pos < (s["lens"] - s["new"])[:, None])
    weights = s["weights"].flatten().clone()
    weights[slot[inside]] = (old + add)[inside]
    return weights.view(s["weights"].shape)


def _quantized(x):
    """fp32 [..., dim] -> codes [..., dim / 32, 32], scales"""
    f = x.unflatten(-1, (-1, 32))
    a = f.abs()
    scale = _cut(a.amax(-1, keepdim=True).clamp(min=1e-8) / 6.0)
    # the nearest value, a tie to the even code: the products are exact in 32 bits
    code = ((a > 0.25 * scale).to(torch.uint8) + (a >= 0.75 * scale) + (a > 1.25 * scale) + (a >= 1.75 * scale)
            + (a > 2.5 * scale) + (a >= 3.5 * scale) + (a > 5.0 * scale))
    return code + 8 * ((f < 0) & (code > 0)), scale.squeeze(-1).to(torch.bfloat16)


def _write(s):
    kc, ks, vc, vs = s["cache"]
    n, h, size, half = kc.shape
    keep = s["slots"] >= 0
    # (rows without a slot go to the block that no slot reaches)
    slot = torch.where(keep, s["slots"], (n - 1) * size)
    at, head = (slot // size)[:, None], torch.arange(h, device=slot.device)
    place = (slot % size)[:, None]
    dc = half // 16
    pair = torch.tensor([1, 16], dtype=torch.uint8, device=slot.device)
    code, scale = _quantized(s["k"].float())
    # [rows, heads, chunk, eighth of it, pair, half]
    byte = (code.view(-1, h, dc, 4, 4, 2) * pair).sum(-1).to(torch.uint8)
    kc[at, head, place] = byte.transpose(2, 3).reshape(-1, h, half)
    ks[at, head, place] = scale
    code, scale = _quantized(s["v"].float())
    # [rows, heads, pair of sixteens, half, dim of the sixteen]
    byte = (code.view(-1, h, dc, 2, 16) * pair[:, None]).sum(3).to(torch.uint8)
    tiles = vc.view(n, h, size // 16, 4, 16, 4, dc)
    tiles[at, head, place // 16, place % 16 // 4, :, place % 4] = byte.transpose(2, 3)
    vs[at, head, place] = scale
    k, v = _dense_k(kc, ks), _dense_v(vc, vs)
    return tuple((x.flatten(0, 1)[slot] * keep[:, None, None]).to(s["dtype"]) for x in (k, v))


def _evict(s):
    lens, most, context = s["lens"].long(), s["most"], s["context"]
    pos = torch.arange(context, device=lens.device)
    inside = pos < lens[:, None]
    slot = s["tables"].long()[:, pos // s["block"]] * s["block"] + pos % s["block"]
    weight = s["weights"].flatten()[slot.clamp(min=0)]
    kept = lens.clamp(max=most)
    # first the sinks, then the newest tokens, then by weight; of equal ones the lower index
    sink = pos < min(s["sinks"], most)
    recent = (pos >= (lens - min(s["recent"], max(most - s["sinks"], 0)))[:, None]) & inside
    rank = torch.where(sink | recent, float("inf"), weight).masked_fill(~inside, -1.0)
    order = rank.sort(stable=True, dim=-1, descending=True).indices[:, :most]
    # (beyond the kept ones, of a request that is shorter than the budget, nothing moves)
    live = torch.arange(order.shape[1], device=lens.device) < kept[:, None]
    order = order.masked_fill(~live, context).sort(-1).values
    source, target = slot.gather(1, order.clamp(max=context - 1))[live], slot[:, :order.shape[1]][live]
    weights = s["weights"].flatten().clone()
    weights[target] = weights[source]
    return kept.to(torch.int32), weights.view(s["weights"].shape), [_moved(c, s, source, target) for c in s["layers"]]


def _moved(cache, s, source, target):
    if s["bits"] == 16:
        return [_moved_rows(c.flatten(0, 1).clone(), source, target).view(c.shape) for c in cache]
    kc, ks, vc, vs = cache
    n, h, size, half = kc.shape

    # each as [slots, heads, ...], and back
    def by_row(x):
        return _moved_rows(x.transpose(1, 2).reshape(n * size, h, -1), source, target).view(n, size, h, -1).transpose(1, 2)

    tiles = vc.view(n, h, size // 16, 4, 16, 4, half // 16).permute(0, 2, 3, 5, 1, 4, 6).reshape(n * size, h, 16, -1)
    tiles = _moved_rows(tiles, source, target).view(n, size // 16, 4, 4, h, 16, half // 16).permute(0, 4, 1, 2, 5, 3, 6)
    k, v = _dense_k(by_row(kc), by_row(ks)), _dense_v(tiles.reshape(vc.shape), by_row(vs))
    return [x.flatten(0, 1).to(torch.bfloat16) for x in (k, v)]


def _moved_rows(rows, source, target):
    rows[target] = rows[source]
    return rows


# ---------------------------------------------------------------------------
# work and definition
# ---------------------------------------------------------------------------

def _sizes(case):
    """rows and tokens of the requests, as prepare spreads them (not which goes with which)"""
    t, n, context = case["tokens"], case["requests"], case["context"]
    rows = _even((t + 1) // 2, t, n)
    return [(r, max(r, c)) for r, c in zip(rows, _even((context + 1) // 2, context, n))]


def _row_bytes(case):
    _, kv, dim = MODELS[case["model"]]
    return kv * dim * 2 if case["bits"] == 16 else kv * (dim // 2 + dim // 16)


def work(case):
    kind, (heads, kv, dim) = case["kind"], MODELS[case["model"]]
    if kind == "write":
        rows = case["rows"] * case["keep"]
        return {"bytes": int(case["rows"] * 8 + rows * kv * 2 * (4 * dim + 2 * (dim // 2 + dim // 16))), "flops": 0}
    if kind == "evict":
        n, context, most = case["requests"], case["context"], case["budget"]
        lens = _even((context * 3 + 3) // 4, context, n)
        pool = sum((x + case["block"] - 1) // case["block"] for x in lens) * case["block"]
        # the clone of the caches, the kept rows read and written where some token goes
        moved = sum(most for x in lens if x > most)
        rows = 4 * case["layers"] * _row_bytes(case) * (pool + moved)
        return {"bytes": rows + 8 * pool + 8 * moved + 4 * sum(lens), "flops": 0}
    pairs = keys = 0
    window, sinks = case["window"], case["sinks"]
    for rows, length in _sizes(case):
        if not window:
            pairs += rows * (length - rows) + rows * (rows + 1) // 2
            keys += length
            continue
        first = length - rows  # the first row's place
        ends = [p + 1 - max(0, p + 1 - window) for p in range(first, length)]
        extra = [min(sinks, max(0, p + 1 - window)) for p in range(first, length)]
        pairs += sum(ends) + sum(extra)
        low = max(0, first + 1 - window)
        keys += length - low + min(sinks, low)
    rows = sum(r for r, _ in _sizes(case))
    if kind == "weigh":
        total = sum(x for _, x in _sizes(case))
        return {"bytes": keys * _row_bytes(case) + rows * heads * (2 * dim + 4) + 8 * total, "flops": 2 * dim * heads * pairs}
    return {"bytes": 2 * keys * _row_bytes(case) + rows * heads * (4 * dim + (4 if case["lse"] else 0)),
            "flops": 4 * dim * heads * pairs}


def exact(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    if case["kind"] == "write":
        keep = s["slots"] >= 0
        return tuple(_exact_rows(s[x].double()) * keep[:, None, None] for x in "kv")
    if case["kind"] == "evict":
        return _exact_evict(s)
    return _exact_attend(s) if case["kind"] == "attend" else _exact_weigh(s)


def _exact_rows(x):
    out = torch.empty_like(x)
    value = torch.tensor(VALUES, dtype=torch.float64, device="cuda")
    for first in range(0, x.shape[-1], 32):
        part = x[..., first:first + 32]
        # the scale that is stored: the quotient in 32 bits, its first 6 significant bits
        scale = part.abs().max(-1).values.float().clamp(min=1e-8) / 6
        mantissa, power = torch.frexp(scale)
        scale = torch.ldexp(torch.floor(mantissa * 64) / 64, power).double()
        far = (part.abs()[..., None] - value * scale[..., None, None]).abs()
        near = far.min(-1, keepdim=True).values
        # (of two at the same distance, the even code)
        code = torch.where(far == near, torch.arange(8, device="cuda") + 8 * (torch.arange(8, device="cuda") % 2), 99)
        out[..., first:first + 32] = value[code.min(-1).values % 8] * scale[..., None] * part.sign()
    return out


def _exact_unpacked(codes, scale, values):
    """A 4-bit cache's keys or values in 64 bits, [blocks * block_size, kv_heads, head_dim], dim by dim."""
    n, h, size, half = codes.shape
    dim, dc = 2 * half, half // 16
    token = torch.arange(size, device="cuda")
    out = torch.empty((n, size, h, dim), dtype=torch.float64, device="cuda")
    table = torch.tensor(VALUES + tuple(-x for x in VALUES), dtype=torch.float64, device="cuda")
    flat = codes.reshape(n, h, -1)
    for d in range(dim):
        if values:
            byte = token // 16 * 16 * half + ((token % 16 // 4 * 16 + d % 16) * 4 + token % 4) * dc + d // 32
            high = d // 16 % 2
        else:
            byte = token * half + 4 * (d % 32 // 8 * dc + d // 32) + d % 8 // 2
            high = d % 2
        out[..., d] = (table[(flat[:, :, byte] >> (4 * high) & 15).long()] * scale[..., d // 32].double()).transpose(1, 2)
    return out.flatten(0, 1)


def _exact_parts(s):
    """For each request and key head: rows' places in the batch, its heads, scores in 64 bits with -inf, its slots."""
    heads, dim = s["q"].shape[1:]
    keys = _exact_unpacked(*s["cache"][:2], False) if s["bits"] == 4 else s["cache"][0].flatten(0, 1)
    per = heads // keys.shape[1]
    lens, offsets = s["lens"].tolist(), s["offsets"].tolist()
    for b, length in enumerate(lens):
        lo, hi = offsets[b], offsets[b + 1]
        j = torch.arange(length, device="cuda")
        slots = s["tables"][b].long()[j // s["block"]] * s["block"] + j % s["block"]
        place = torch.arange(length - (hi - lo), length, device="cuda")[:, None]
        hidden = j > place
        if s["window"]:
            hidden |= (j <= place - s["window"]) & (j >= s["sinks"])
        for h in range(keys.shape[1]):
            k = keys[slots, h].double()
            for g in range(h * per, (h + 1) * per):
                logit = s["q"][lo:hi, g].double() @ k.t() / dim ** 0.5
                yield lo, hi, h, g, logit.masked_fill_(hidden, float("-inf")), slots


def _exact_attend(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    values = _exact_unpacked(*s["cache"][2:], True) if s["bits"] == 4 else s["cache"][1].flatten(0, 1)
    for lo, hi, h, g, logit, slots in _exact_parts(s):
        lse[lo:hi, g] = torch.logsumexp(logit, 1)
        out[lo:hi, g] = torch.nan_to_num(torch.softmax(logit, 1)) @ values[slots, h].double()
    return (out, lse) if s["lse"] else out


def _exact_weigh(s):
    weights = s["weights"].double().flatten()
    fresh = set()
    lens, new = s["lens"].tolist(), s["new"].tolist()
    for lo, hi, _, g, logit, slots in _exact_parts(s):
        if lo not in fresh:
            fresh.add(lo)
            weights[slots[len(slots) - (hi - lo):]] = 0
        weights[slots] += torch.exp(logit - s["lse"][lo:hi, g].double()[:, None]).sum(0)
    assert len(fresh) == len(lens) == len(new)
    return weights.view(s["weights"].shape)


def _exact_evict(s):
    kept, weights, block = [], s["weights"].double().flatten(), s["block"]
    moves = []
    for b, length in enumerate(s["lens"].tolist()):
        most = s["most"]
        if length <= most:
            kept.append(length)
            continue
        slot = [int(x) * block + i for x in s["tables"][b].tolist() for i in range(block)][:length]
        w = s["weights"].flatten()[torch.tensor(slot, device="cuda")].tolist()
        sinks = min(s["sinks"], most)
        recent = min(s["recent"], most - sinks)
        others = sorted(range(sinks, length - recent), key=lambda i: (-w[i], i))[:most - sinks - recent]
        stay = list(range(sinks)) + sorted(others) + list(range(length - recent, length))
        moves += [(slot[i], slot[j]) for j, i in enumerate(stay)]
        kept.append(most)
    source, target = torch.tensor(moves, dtype=torch.long, device="cuda").reshape(-1, 2).t()
    weights[target] = weights[source]
    layers = None
    if s["bits"] == 16:
        layers = [[c.double().flatten(0, 1).index_copy(0, target, c.double().flatten(0, 1)[source]).view(c.shape) for c in x]
                  for x in s["layers"]]
    return torch.tensor(kept, dtype=torch.int32, device="cuda"), weights.view(s["weights"].shape), layers
