"""Operators of speculative decoding over a paged cache, as measurable cases.

A serving step that drafts tokens with 4-bit weights and verifies a tree of them
against the cache of a request runs, through ``pageserve_amd``:

``append``    block tables extended by the requests' new tokens, and the slot
              of every row (``append_blocks``).
``write``     key and value rows stored at their slots (``write_kv``).
``attend``    attention of each request's drafted tokens over its cached tokens
              and their own ancestors (``tree_attention``).
``quantize``  a weight brought to 4-bit codes with one scale per group of
              columns, and its dense values (``QuantizedWeight4``).
``linear``    a projection of a few tokens with such a weight (``linear4``).

Sizes are those of the models this repository serves: the 2048-hidden,
11008-wide model with 16 query and 2 key heads of 128 ("3b"), the 896-hidden,
4864-wide one with 14 query and 2 key heads of 64 ("0.5b"), a vocabulary of
151936, and cache blocks of 16 tokens and more.

With ``own`` false the operators are computed in elementary torch operations,
in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import torch

own = False

#        hidden, intermediate, query heads, key heads, head_dim
MODELS = {"3b": (2048, 11008, 16, 2, 128), "0.5b": (896, 4864, 14, 2, 64)}
VOCAB = 151936
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
#: the values of the 4-bit codes 0..7 (code + 8 is the negative value)
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # after a verification step of eight users: 12 drafted rows each, a few of them accepted
        {"name": "append-accepted-8", "kind": "append", "requests": 8, "tokens": 12, "block": 16, "accept": True},
        # prompts of 64 requests admitted at once
        {"name": "append-prompts-64", "kind": "append", "requests": 64, "tokens": 400, "block": 16, "accept": False},
        # the accepted rows of one layer stored, the rejected ones left out
        {"name": "write-accepted-96", "kind": "write", "model": "3b", "rows": 96, "dtype": "bf16", "block": 16,
         "keep": 0.4},
        # a chunk of prompts stored, all rows
        {"name": "write-prompts-8192", "kind": "write", "model": "3b", "rows": 8192, "dtype": "f16", "block": 64,
         "keep": 1.0},
        # plain decoding, one token of each of six short chats
        {"name": "attend-step-6", "kind": "attend", "model": "0.5b", "requests": 6, "tokens": 1, "context": 700,
         "block": 16, "dtype": "bf16"},
        # trees of up to 24 tokens over two very long documents
        {"name": "attend-long-2", "kind": "attend", "model": "3b", "requests": 2, "tokens": 24, "context": 120000,
         "block": 16, "dtype": "bf16"},
        # the widest trees of a full batch
        {"name": "attend-wide-24", "kind": "attend", "model": "3b", "requests": 24, "tokens": 64, "context": 8000,
         "block": 64, "dtype": "f16"},
        # one small projection of a bf16 checkpoint
        {"name": "quantize-0.5b-v", "kind": "quantize", "rows": 128, "cols": 896, "group": 32, "dtype": "bf16"},
        # the largest projection of an fp32 checkpoint
        {"name": "quantize-3b-gate", "kind": "quantize", "rows": 11008, "cols": 2048, "group": 128, "dtype": "f32"},
        # one drafted token through the widest projection
        {"name": "linear-3b-gate-1", "kind": "linear", "rows": 11008, "cols": 2048, "group": 128, "tokens": 1,
         "bias": False, "residual": False, "out": "bf16"},
        # five tokens through the long one, added to the residual stream
        {"name": "linear-3b-down-5", "kind": "linear", "rows": 2048, "cols": 11008, "group": 64, "tokens": 5,
         "bias": False, "residual": True, "out": "bf16"},
        # the logits of a batch of drafts
        {"name": "linear-head-30", "kind": "linear", "rows": VOCAB, "cols": 2048, "group": 32, "tokens": 30,
         "bias": False, "residual": False, "out": "f32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["append", "write", "attend", "attend", "attend", "quantize", "linear", "linear", "linear"])
    model = rng.choice(["3b", "3b", "0.5b"])
    block = rng.choice([16, 16, 32, 64, 128])
    if kind == "append":
        accept = rng.random() < 0.5
        return {"kind": kind, "requests": _log_int(rng, 1, 400), "tokens": _log_int(rng, 1, 64 if accept else 500),
                "block": block, "accept": accept}
    if kind == "write":
        return {"kind": kind, "model": model, "rows": _log_int(rng, 1, 8192), "dtype": rng.choice(["bf16", "f16"]),
                "block": block, "keep": rng.choice([0.3, 0.8, 1.0])}
    if kind == "attend":
        tokens, requests = rng.choice([1, rng.randint(2, 16), rng.randint(17, 64)]), _log_int(rng, 1, 48)
        # (as much as the largest listed case at most)
        most = min(120000, 12_000_000 // (tokens * requests), 240_000 // requests)
        return {"kind": kind, "model": model, "requests": requests, "tokens": tokens,
                "context": _log_int(rng, 1, most), "block": block, "dtype": rng.choice(["bf16", "bf16", "f16"])}
    hidden, inter, heads, kv, dim = MODELS[model]
    rows, cols = rng.choice([(hidden, hidden), (kv * dim, hidden), (inter, hidden), (hidden, inter),
                             (_log_int(rng, 8, 16384), 16 * _log_int(rng, 4, 700))])
    group = rng.choice([32, 64, 128])
    if kind == "quantize":
        rows = min(rows, 22_500_000 // cols)
        return {"kind": kind, "rows": rows, "cols": cols, "group": group, "dtype": rng.choice(["bf16", "f32"])}
    out = rng.choice(["bf16", "bf16", "f32"])
    return {"kind": kind, "rows": rows, "cols": cols, "group": group,
            "tokens": rng.choice([1, 1, _log_int(rng, 1, 16), _log_int(rng, 1, 64)]), "bias": rng.random() < 0.4,
            "residual": out == "bf16" and rng.random() < 0.4, "out": out}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _spread(gen, lo, hi, n):
    """n numbers spread evenly over lo..hi, in random order, int32"""
    return torch.tensor(_even(lo, hi, n), dtype=torch.int32, device="cuda")[
        torch.randperm(n, generator=gen, device="cuda")]


def _even(lo, hi, n):
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _offsets(counts):
    """[0, c0, c0 + c1, ...] int32"""
    return torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)


def _tables(gen, blocks, columns, pool):
    """Distinct random block ids in each request's first ``blocks`` columns, -1
    behind, and the ids of the pool left over, in random order."""
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    first = _offsets(blocks)[:-1, None]
    col = torch.arange(columns, device="cuda")
    inside = col < blocks[:, None]
    at = (first + col).clamp(max=pool - 1)
    return torch.where(inside, order[at.long()], -1).to(torch.int32), order[int(blocks.sum()):]


def _append_inputs(case, seed):
    gen, n, t, s = _gen(seed), case["requests"], case["tokens"], case["block"]
    rows = _spread(gen, (t + 1) // 2, t, n)
    lens = _spread(gen, 0, 2000, n)
    offsets = _offsets(rows)
    total = int(offsets[-1])
    new, index = rows, None
    if case["accept"]:
        # each request keeps the first rows of a path: row k of it, or -1
        keep = torch.rand(total, generator=gen, device="cuda") < 0.3
        before = keep.cumsum(0) - keep.long()
        owner = torch.searchsorted(offsets[1:].contiguous(), torch.arange(total, device="cuda"), right=True)
        rank = before - before[offsets[:-1].long()][owner]
        index = torch.where(keep, rank, -1).to(torch.int32)
        new = torch.zeros(n, dtype=torch.int64, device="cuda").index_add_(0, owner, keep.long()).to(torch.int32)
    have = (lens + s - 1) // s
    columns = (2000 + t + s - 1) // s
    used = int(have.sum())
    # the pool is nearly as full as a busy server's
    pool = used + n * (t // s + 1) + 1
    tables, left = _tables(gen, have, columns, pool)
    free = torch.zeros(pool, dtype=torch.int32, device="cuda")
    free[:left.numel()] = left
    # lens, the count of free blocks and the tables in one buffer, as a server that copies its state would hold them
    state = torch.cat([lens, torch.tensor([left.numel()], dtype=torch.int32, device="cuda"), tables.reshape(-1)])
    return {"state": state, "requests": n, "columns": columns, "new": new, "offsets": offsets, "free": free,
            "index": index, "block": s, "rows": total}


def _write_inputs(case, seed):
    gen, n, s = _gen(seed), case["rows"], case["block"]
    _, _, _, kv, dim = MODELS[case["model"]]
    dt = DTYPES[case["dtype"]]
    blocks = (n + s - 1) // s + 4
    slots = torch.randperm(blocks * s, generator=gen, device="cuda")[:n]
    if case["keep"] < 1:
        slots = torch.where(torch.rand(n, generator=gen, device="cuda") < case["keep"], slots, -1)
    else:  # a prompt's rows fill whole blocks
        base = torch.randperm(blocks, generator=gen, device="cuda")
        at = torch.arange(n, device="cuda")
        slots = base[at // s] * s + at % s
    return {"k": _randn(gen, n, kv, dim, dtype=dt), "v": _randn(gen, n, kv, dim, dtype=dt),
            "k_cache": _randn(gen, blocks, s, kv, dim, dtype=dt), "v_cache": _randn(gen, blocks, s, kv, dim, dtype=dt),
            "slots": slots}


def _attend_inputs(case, seed):
    gen, n, t, s = _gen(seed), case["requests"], case["tokens"], case["block"]
    _, _, heads, kv, dim = MODELS[case["model"]]
    dt = DTYPES[case["dtype"]]
    rows = _spread(gen, (t + 1) // 2, t, n)
    lens = _spread(gen, case["context"] // 2, case["context"], n)
    offsets = _offsets(rows)
    total = int(offsets[-1])
    # parents: some earlier token of the request, often the one before; roots now and then
    local = torch.arange(total, device="cuda") - offsets[:-1].long().repeat_interleave(rows.long())
    back = (torch.rand(total, generator=gen, device="cuda") ** 2 * 4).long() + 1
    parents = (local - back).clamp(min=-1).to(torch.int32)
    have = (lens + s - 1) // s
    columns = (case["context"] + s - 1) // s
    pool = int(have.sum()) + 3
    tables, _ = _tables(gen, have, columns, pool)
    return {"q": _randn(gen, total, heads, dim, dtype=dt), "k": _randn(gen, total, kv, dim, dtype=dt),
            "v": _randn(gen, total, kv, dim, dtype=dt), "k_cache": _randn(gen, pool, s, kv, dim, dtype=dt),
            "v_cache": _randn(gen, pool, s, kv, dim, dtype=dt), "tables": tables, "lens": lens, "offsets": offsets,
            "parents": parents, "tokens": t, "context": case["context"]}


def _linear_inputs(case, seed):
    gen, n, k, m = _gen(seed), case["rows"], case["cols"], case["tokens"]
    codes, scale = _quantize(_randn(gen, n, k, std=0.02), case["group"])
    return {"codes": codes, "scale": scale, "group": case["group"], "x": _randn(gen, m, k),
            "bias": _randn(gen, n, std=0.1) if case["bias"] else None,
            "residual": _randn(gen, m, n) if case["residual"] else None, "out": DTYPES[case["out"]]}


def _inputs(case, seed):
    kind = case["kind"]
    if kind == "append":
        return _append_inputs(case, seed)
    if kind == "write":
        return _write_inputs(case, seed)
    if kind == "attend":
        return _attend_inputs(case, seed)
    if kind == "linear":
        return _linear_inputs(case, seed)
    return {"w": _randn(_gen(seed), case["rows"], case["cols"], std=0.02, dtype=DTYPES[case["dtype"]]),
            "group": case["group"]}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["kind"] = case["kind"]
    if own and case["kind"] == "linear":
        # the weight in the layout that the program keeps it in
        from pageserve_amd import QuantizedWeight4

        state["weight"] = QuantizedWeight4.from_codes(state["codes"], state["scale"], case["group"], torch.bfloat16)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "append":
        return _append(state)
    if kind == "write":
        return _write(state)
    if kind == "attend":
        return _attend(state)
    if kind == "linear":
        return _linear(state)
    codes, scale = _quantize(state["w"], state["group"])
    return _dense(codes, scale, state["group"]).to(state["w"].dtype), scale


def _views(s):
    """A copy of the paged state, as (lens, free count, tables)."""
    buf, n = s["state"].clone(), s["requests"]
    return buf[:n], buf[n:n + 1], buf[n + 1:].view(n, s["columns"])


def _run_own(s):
    import pageserve_amd as P

    kind = s["kind"]
    if kind == "append":
        lens, count, tables = _views(s)
        slots, status = P.append_blocks(lens, s["new"], s["offsets"], tables, s["free"], count, s["block"], s["rows"],
                                        index=s["index"])
        return slots, status, lens, count, tables
    if kind == "write":
        P.write_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return s["k_cache"], s["v_cache"]
    if kind == "attend":
        return P.tree_attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"],
                                s["offsets"], s["parents"], max_tokens=s["tokens"], max_context=s["context"])
    if kind == "linear":
        return P.linear4(s["x"], s["weight"], s["bias"], out_dtype=s["out"], residual=s["residual"])
    w = P.QuantizedWeight4(s["w"], s["group"])
    return w.dense(), w.scale


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _append(s):
    lens, count, tables = _views(s)
    bs, new, offsets = s["block"], s["new"], s["offsets"]
    have, want = (lens + bs - 1) // bs, (lens + new + bs - 1) // bs
    fits = want <= tables.shape[1]
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= count))
    status = torch.where(served, 0, torch.where(fits, 1, 2)).to(torch.int32)
    # the new table entries, taken from the end of the free list in request order
    col = torch.arange(tables.shape[1], device=lens.device)
    fresh = served[:, None] & (col >= have[:, None]) & (col < want[:, None])
    entry = (upto - need)[:, None] + col - have[:, None]
    pick = (count.long() - 1 - entry).clamp(0, s["free"].numel() - 1)
    tables.copy_(torch.where(fresh, s["free"][pick], tables))
    # the rows' slots
    row = torch.arange(s["rows"], device=lens.device)
    owner = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=lens.numel() - 1)
    index = s["index"].long() if s["index"] is not None else row - offsets[owner]
    pos = (lens[owner] + index).clamp(min=0)
    block = tables[owner, (pos // bs).clamp(max=tables.shape[1] - 1)].long()
    inside = served[owner] & (index >= 0) & (index < new[owner]) & (block >= 0) & (row < offsets[-1])
    slots = torch.where(inside, block * bs + pos % bs, -1)
    lens.add_(torch.where(served, new, 0))
    count.sub_(torch.where(served, need, 0).sum().to(torch.int32))
    return slots, status, lens, count, tables


def _write(s):
    # (a row without a slot stores the first kept row once more; where none is kept, the last slot its own values)
    keep = s["slots"] >= 0
    row = torch.where(keep, torch.arange(keep.numel(), device=keep.device), keep.int().argmax())
    at = s["slots"][row]
    some = (at >= 0)[:, None, None]
    kc, vc = s["k_cache"].flatten(0, 1), s["v_cache"].flatten(0, 1)
    kc[at] = torch.where(some, s["k"][row], kc[at])
    vc[at] = torch.where(some, s["v"][row], vc[at])
    return s["k_cache"], s["v_cache"]


def _attend(s):
    q, k, v, lens, offsets = s["q"], s["k"], s["v"], s["lens"].long(), s["offsets"].long()
    (total, heads, dim), kv, n, t = q.shape, k.shape[1], lens.numel(), s["tokens"]
    bs = s["k_cache"].shape[1]
    dev = q.device
    # every request's rows and cached tokens, padded to the longest
    token = torch.arange(t, device=dev)
    rows = offsets[:-1, None] + token
    live = rows < offsets[1:, None]
    rows = rows.clamp(max=total - 1)
    pos = torch.arange(s["context"], device=dev)
    cached = pos < lens[:, None]
    slot = (s["tables"].long().clamp(min=0)[:, pos // bs] * bs + pos % bs) * cached
    kc = s["k_cache"].flatten(0, 1)[slot].float().permute(0, 2, 1, 3)  # [n, kv, context, dim]
    vc = s["v_cache"].flatten(0, 1)[slot].float().permute(0, 2, 1, 3)
    kt, vt = (x[rows].float().permute(0, 2, 1, 3) for x in (k, v))      # [n, kv, t, dim]
    qt = q[rows].float().view(n, t, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)  # [n, kv, group, t, dim]
    # which drafted tokens a token sees: itself and its ancestors
    parent = s["parents"].long()[rows]
    step = (parent[:, :, None] == token) & live[:, :, None]
    sees = torch.linalg.matrix_power(torch.eye(t, device=dev) + step.float(), max(t, 1)) > 0
    qf = qt.reshape(n, kv, -1, dim)
    keys = torch.cat([kc, kt], 2)
    score = torch.matmul(qf, keys.transpose(2, 3).contiguous()) * dim ** -0.5
    score = score.view(n, kv, heads // kv, t, -1)
    seen = torch.cat([cached[:, None, :].expand(n, t, -1), sees & live[:, None, :]], 2)
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kv, -1, p.shape[-1]), torch.cat([vc, vt], 2))
    o = o.view(n, kv, heads // kv, t, dim).permute(0, 3, 1, 2, 4).reshape(n, t, heads, dim)
    return o[live].to(q.dtype)


def _quantize(w, group):
    n, k = w.shape
    pad = -k % group
    f = torch.nn.functional.pad(w.float(), (0, pad)).view(n, -1, group)
    a = f.abs()
    scale = (a.amax(2, keepdim=True).clamp(min=1e-8) / 6.0).to(torch.bfloat16)
    s = scale.float()
    # the nearest value, a tie to the even code: the products are exact in 32 bits
    code = ((a > 0.25 * s).to(torch.uint8) + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s) + (a > 2.5 * s)
            + (a >= 3.5 * s) + (a > 5.0 * s))
    code = code + 8 * ((f < 0) & (code > 0))
    return code.view(n, -1)[:, :k].contiguous(), scale.squeeze(2)


def _dense(codes, scale, group):
    value = torch.tensor(VALUES + tuple(-x for x in VALUES), device=codes.device)
    n, k = codes.shape
    per = scale.float().repeat_interleave(group, 1)[:, :k]
    return value[codes.int()] * per


def _linear(s):
    y = torch.matmul(s["x"].float(), _dense(s["codes"], s["scale"], s["group"]).t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["residual"] is not None:
        # the projection is rounded to the output type before it is added, as in the 8-bit linear
        y = y.to(s["out"]).float() + s["residual"].float()
    return y.to(s["out"])


# ---------------------------------------------------------------------------
# work and definition
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "append":
        n, t = case["requests"], case["tokens"]
        rows = sum(_even((t + 1) // 2, t, n))
        columns = (2000 + t + case["block"] - 1) // case["block"]
        # state copied (read and written), index read, slots written
        return {"bytes": 8 * (n * (columns + 4)) + rows * (12 if case["accept"] else 8), "flops": 0}
    if kind == "write":
        _, _, _, kv, dim = MODELS[case["model"]]
        return {"bytes": int(case["rows"] * (8 + case["keep"] * 8 * kv * dim)), "flops": 0}
    if kind == "attend":
        _, _, heads, kv, dim = MODELS[case["model"]]
        n, t, length = case["requests"], case["tokens"], case["context"]
        tokens = sum(_even((t + 1) // 2, t, n))
        length = sum(_even(length // 2, length, n))
        pairs = tokens * (length // n + 1)
        return {"bytes": 4 * dim * (length * kv + tokens * (heads + kv)), "flops": 4 * dim * heads * pairs}
    n, k = case["rows"], case["cols"]
    packed = n * k // 2 + n * ((k + case["group"] - 1) // case["group"]) * 2
    if kind == "quantize":
        wide = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * n * k * wide + 2 * packed, "flops": 0}
    m = case["tokens"]
    return {"bytes": packed + 2 * m * k + m * n * (4 if case["out"] == "f32" else 2)
            + (2 * m * n if case["residual"] else 0) + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "append":
        return None
    if kind == "write":
        out = []
        for rows, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
            flat = cache.double().flatten(0, 1)
            keep = (s["slots"] >= 0).nonzero().squeeze(1)
            flat.index_copy_(0, s["slots"][keep], rows.double()[keep])
            out.append(flat.view(cache.shape))
        return tuple(out)
    if kind == "attend":
        return _exact_attend(s)
    if kind == "quantize":
        return _exact_quantize(s["w"].double(), s["group"])
    table = torch.tensor([(-1) ** (c // 8) * VALUES[c % 8] for c in range(16)], dtype=torch.float64, device="cuda")
    y = []
    for first in range(0, case["rows"], 16384):  # a slice of output columns at a time
        codes, scale = s["codes"][first:first + 16384].long(), s["scale"][first:first + 16384].double()
        at = torch.arange(case["cols"], device="cuda") // case["group"]
        y.append(s["x"].double() @ (table[codes] * scale[:, at]).t())
    y = torch.cat(y, 1)
    if s["bias"] is not None:
        y = y + s["bias"].double()
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_attend(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    heads, dim = s["q"].shape[1:]
    per = heads // s["k"].shape[1]
    bs = s["k_cache"].shape[1]
    lens, offsets, parents = s["lens"].tolist(), s["offsets"].tolist(), s["parents"].tolist()
    for b, length in enumerate(lens):
        lo, hi = offsets[b], offsets[b + 1]
        blocks = s["tables"][b, :(length + bs - 1) // bs].long()
        see = torch.zeros(hi - lo, length + hi - lo, dtype=torch.bool, device="cpu")
        see[:, :length] = True
        for i in range(hi - lo):
            j = i
            while j >= 0:
                see[i, length + j] = True
                j = parents[lo + j]
        see = see.to("cuda")
        for h in range(s["k"].shape[1]):
            key = torch.cat([s["k_cache"][blocks, :, h].reshape(-1, dim)[:length], s["k"][lo:hi, h]]).double()
            val = torch.cat([s["v_cache"][blocks, :, h].reshape(-1, dim)[:length], s["v"][lo:hi, h]]).double()
            for g in range(h * per, (h + 1) * per):
                logit = s["q"][lo:hi, g].double() @ key.t() / dim ** 0.5
                out[lo:hi, g] = torch.softmax(logit.masked_fill(~see, float("-inf")), 1) @ val
    return out


def _exact_quantize(w, group):
    n, k = w.shape
    value = torch.tensor(VALUES, dtype=torch.float64, device="cuda")
    dense, scales = torch.empty_like(w), []
    for first in range(0, k, group):
        part = w[:, first:first + group]
        # the scale that is stored: the quotient in 32 bits, then in 16
        scale = (part.abs().max(1).values.float().clamp(min=1e-8) / 6).bfloat16().double()
        far = (part.abs()[:, :, None] - value * scale[:, None, None]).abs()
        near = far.min(2, keepdim=True).values
        # (of two at the same distance, the even code)
        code = torch.where(far == near, torch.arange(8, device="cuda") + 8 * (torch.arange(8, device="cuda") % 2), 99)
        dense[:, first:first + group] = value[code.min(2).values % 8] * scale[:, None] * part.sign()
        scales.append(scale)
    return dense, torch.stack(scales, 1)
