"""Attention over windows, accumulated weights and eviction where a call is unlike the plain
one: other strides and layouts, rows outside of every request, numbers that are not finite,
streams, graphs, tables and caches beyond 32 bits, refusals (tests/bounded.py: the bounds)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bounded import HEADS, Batch
from oracle import window_oracle as W
from pageserve_amd import KVCache4, accumulate_weights, evict_tokens, window_attention, window_attention4, write_kv4

pytestmark = pytest.mark.gpu


def attend(b, args, many=False, **kw):
    """many: with as many rows of no request behind them as make the batch one of many rows"""
    call = window_attention4 if b.bits == 4 else window_attention
    if not many:
        return call(*args, **kw)
    rows, out = args[0].shape[0], kw.pop("out", None)
    q = torch.nn.functional.pad(args[0], (0, 0, 0, 0, 0, 40000))
    full = torch.full_like(q, 11.0)
    if out is not None:
        full[:rows] = out
    got = call(q, *args[1:], out=full, **kw)
    assert (full[rows:] == 11.0).all()
    if out is not None:
        out.copy_(full[:rows])
    return (got[0][:rows], got[1][:rows]) if isinstance(got, tuple) else got[:rows]


def batch(tokens, bits, dtype=torch.bfloat16, heads=(16, 2, 128), **kw):
    """Requests with some, one, no and (last) more rows than tokens"""
    lens, counts = [tokens + 100, 200, 40, 90, max(1, tokens // 2)], [tokens, 1, 0, min(tokens, 7), tokens]
    return Batch(tokens, lens, counts, *heads, 16, dtype, bits, **kw)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [1, 3, 20, 80, 1500])
def test_rows_of_a_fused_projection_and_rows_of_no_request(gpu, tokens, bits):
    b = batch(tokens, bits, pad=5)
    q, *rest = b.args(gpu)
    fused = torch.full((q.shape[0], 20, 128), float("nan"), dtype=q.dtype, device=gpu)
    fused[:, 2:18] = q
    out = torch.full_like(q, 7.0)
    want = b.oracle(window=60, sinks=3)
    got = attend(b, [fused[:, 2:18], *rest], window=60, sinks=3, return_lse=True, out=out)
    assert got[0].data_ptr() == out.data_ptr() and (out[-5:] == 7.0).all()
    b.check(got, want)
    # in place
    attend(b, [q, *rest], window=60, sinks=3, out=q)
    b.check(q, want)
    assert torch.equal(q[-5:].cpu(), b.q[-5:])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [6, 90, 1000])
def test_rows_beyond_max_tokens_are_left(gpu, tokens, bits):
    b = batch(tokens, bits)
    args = b.args(gpu)
    for most in (1, tokens - 2):
        out = torch.full_like(args[0], -3.0)
        got = attend(b, args, window=50, sinks=1, max_tokens=most, out=out, return_lse=True, max_context=2000)
        want = b.oracle(window=50, sinks=1, max_tokens=most)
        b.check(got, want, f"{most}")
        assert (out[torch.from_numpy(np.isnan(want[1][:, 0])).to(gpu)] == -3.0).all()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("tokens", [1, 70])
def test_caches_of_other_orders(gpu, tokens, many):
    """Heads in front of slots; keys and values in one tensor; both, of one request's own pool"""
    b = batch(tokens, 16, torch.float16, (4, 2, 64))
    q, k, v, *rest = b.args(gpu)
    want = b.oracle(window=70, sinks=2)
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    b.check(attend(b, [q, *turned, *rest], many, window=70, sinks=2, return_lse=True), want)
    both = torch.stack((k, v), 3)
    b.check(attend(b, [q, both[:, :, :, 0], both[:, :, :, 1], *rest], many, window=70, sinks=2, return_lse=True), want)
    halves = torch.cat((k, v), 3)
    b.check(attend(b, [q, halves[..., :64], halves[..., 64:], *rest], many, window=70, sinks=2, return_lse=True), want)
    wide = torch.nn.functional.pad(rest[0], (0, 9), value=1 << 30)
    b.check(attend(b, [q, k, v, wide[:, :rest[0].shape[1]], *rest[1:]], many, window=70, sinks=2, return_lse=True), want)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("tokens", [3, 33, 70, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [16, 4])
def test_batches_of_many_rows(gpu, heads, tokens, dtype, bits):
    lens = [tokens, tokens + 1, 15, 16, 17, 33, 200, 300]
    rng = np.random.default_rng(tokens)
    counts = [tokens, tokens] + [min(int(n), x) for n, x in zip(rng.integers(0, tokens + 1, 4), lens[2:])] + [tokens, 0]
    b = Batch(tokens, lens, counts, *HEADS[heads], 16, dtype, bits, garbage=float("nan"))
    args = b.args(gpu)
    for window, sinks in ((None, 0), (1, 0), (20, 4), (64, 40), (500, 3)):
        kw = {"window": window, "sinks": sinks}
        b.check(attend(b, args, True, return_lse=True, **kw), b.oracle(**kw), f"{kw}")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("context", [3000, 20000])
@pytest.mark.parametrize("tokens", [100, 300])
def test_some_rows_over_a_longer_context(gpu, tokens, context, bits):
    """Either kind of kernel by how many tokens are expected"""
    b = Batch(tokens, [2500, 700], [tokens, 64], 8, 1, 128, 64, torch.bfloat16, bits, garbage=float("inf"))
    args = b.args(gpu)
    for window, sinks in ((None, 0), (900, 70)):
        want = b.oracle(window=window, sinks=sinks)
        b.check(attend(b, args, window=window, sinks=sinks, max_context=context, return_lse=True), want)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [1, 5, 70])
@pytest.mark.parametrize("heads", [(16, 2, 128), (14, 2, 64)])
def test_absent_blocks_and_wrong_numbers_stay_inside(gpu, heads, tokens, bits, many):
    """Blocks that are absent or no numbers of blocks hide their tokens; lengths and offsets are cut to
    what there is."""
    b = batch(tokens, bits, heads=heads)
    b.tables[0, [0, 3, 6]] = -1, 1 << 30, b.blocks
    b.tables[1, :] = -(1 << 31)
    b.tables[3, 2] = -7
    args = b.args(gpu)
    for window, sinks in ((None, 0), (33, 17)):
        want = b.oracle(window=window, sinks=sinks)
        got = attend(b, args, many, window=window, sinks=sinks, return_lse=True)
        assert np.isneginf(want[1]).any()
        b.check(got, want)
        sums = torch.zeros(b.blocks, b.bs, device=gpu)
        lse = torch.nan_to_num(got[1], neginf=0.0)
        accumulate_weights(args[0], args[1], *args[-3:], lse, sums, window=window, sinks=sinks)
        live = float((~torch.isneginf(got[1])).sum())
        assert abs(float(sums.double().sum()) - live) <= live * 2.0 ** -15
    q, *cache, tables, lens, offsets = args
    wild = torch.tensor([(1 << 31) - 1, -5, 1 << 30, 40, -(1 << 31)], dtype=torch.int32, device=gpu)
    out = attend(b, [q, *cache, tables, wild, offsets], many, window=40, sinks=3)
    assert out.shape == q.shape
    turned = torch.tensor([50, -3, (1 << 31) - 1, 2, 1, 0], dtype=torch.int32, device=gpu)
    assert attend(b, [q, *cache, tables, lens, turned], window=40, sinks=3, max_tokens=tokens).shape == q.shape
    sums = torch.zeros(b.blocks, b.bs, device=gpu)
    accumulate_weights(q, cache[0], tables, wild, turned, torch.zeros(q.shape[:2], device=gpu), sums, new_lens=wild)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [5, 24, 90])
@pytest.mark.parametrize("back", [1, 3, 22, 60, 110])
@pytest.mark.parametrize("what", ["inf", "nan", "key"])
@pytest.mark.parametrize("dtype,many", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True),
                                        (torch.float16, True)])
def test_numbers_that_are_not_finite_reach_the_rows_that_see_them(gpu, dtype, many, what, back, tokens, bits):
    heads, kv, dim, window, sinks = 8, 2, 64, 20, 2
    clean = Batch(back, [200, 90], [tokens, 3], heads, kv, dim, 16, dtype, bits)
    want = clean.oracle(window=window, sinks=sinks)
    b = Batch(back, [200, 90], [tokens, 3], heads, kv, dim, 16, dtype, bits)
    blk, at = b.tables[0, (200 - back) // 16], (200 - back) % 16
    if what == "key":
        b.kc[blk, at, 1, 40] = float("nan")
    else:
        b.vc[blk, at, 1, 40] = float(what)
    out, lse = attend(b, b.args(gpu), many, window=window, sinks=sinks, return_lse=True)
    see = torch.from_numpy(W.sees(tokens, 200, window, sinks)[:, 200 - back])
    hit = torch.zeros(out.shape, dtype=torch.bool)
    dims = slice(0, dim) if what == "key" else slice(32, 64) if bits == 4 else slice(40, 41)
    hit[:tokens, heads // kv:, dims] = see[:, None, None]
    bad = ~torch.isfinite(out.cpu())
    assert not bad[~hit].any(), "a row that does not see it"
    sure = hit & (torch.arange(dim) == 40)
    assert bad[sure].all(), "a row that sees it"
    mine = torch.where(hit, torch.from_numpy(want[0]).to(dtype), out.cpu())
    rows = (hit.any(-1) & (what == "key"))
    clean.check((mine, torch.where(rows, torch.from_numpy(want[1]).float(), lse.cpu())), want)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [2, 70])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 400.0, -1e4])
def test_scales(gpu, scale, tokens, bits, many):
    b = batch(tokens, bits, torch.float16, (4, 2, 64))
    args = b.args(gpu)
    want = b.oracle(scale, window=100, sinks=3)
    b.check(attend(b, args, many, window=100, sinks=3, scale=scale, return_lse=True), want)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("requests,tokens", [(700, 1), (300, 66), (513, 3)])
def test_many_requests(gpu, requests, tokens, bits):
    rng = np.random.default_rng(requests)
    lens = rng.integers(1, 90, requests)
    counts = np.minimum(rng.integers(0, tokens + 1, requests), lens).tolist()
    counts[3] = min(tokens, lens[3])
    b = Batch(requests, lens.tolist(), counts, 2, 1, 64, 16, torch.bfloat16, bits, garbage=float("nan"))
    args = b.args(gpu)
    want = b.oracle(window=30, sinks=2)
    b.check(attend(b, args, True, window=30, sinks=2, return_lse=True), want)
    got = attend(b, args, window=30, sinks=2, max_tokens=tokens, return_lse=True)
    b.check(got, want)
    sums = torch.zeros(b.blocks, b.bs, device=gpu)
    accumulate_weights(args[0], args[1], *args[-3:], got[1], sums, window=30, sinks=2)
    live = float((~torch.isneginf(got[1])).sum())
    assert abs(float(sums.double().sum()) - live) <= live * 2.0 ** -15


@pytest.mark.parametrize("tokens", [1, 70])
@pytest.mark.parametrize("bits", [16, 4])
def test_a_cache_beyond_32_bits(gpu, bits, tokens):
    """Blocks whose bytes and elements lie beyond 2^32 and 2^31"""
    b = Batch(9, [tokens + 300, 77], [tokens, 1], 4, 2, 128, 64, torch.bfloat16, bits)
    q, *cache, tables, lens, offsets = b.args(gpu)
    row = 64 * 2 * 128 * 2 if bits == 16 else 64 * 2 * 64
    high = (1 << 32) // row + 100
    args = [q]
    if bits == 16:
        for part in cache:
            big = torch.empty((high + b.blocks, *part.shape[1:]), dtype=part.dtype, device=gpu)
            big[high:] = part
            args.append(big)
    else:
        big = KVCache4(high + b.blocks, 64, 2, 128, gpu)
        slots = torch.arange(b.blocks * 64, device=gpu) + high * 64
        write_kv4(b.kc.to(gpu).flatten(0, 1), b.vc.to(gpu).flatten(0, 1), big, slots)
        args.append(big)
    tables = torch.where(tables >= 0, tables + high, tables)
    want = b.oracle(window=200, sinks=5)
    b.check(attend(b, [*args, tables, lens, offsets], True, window=200, sinks=5, return_lse=True), want)
    out, lse = attend(b, [*args, tables, lens, offsets], window=200, sinks=5, return_lse=True)
    b.check((out, lse), want)
    sums = torch.zeros(high + b.blocks, 64, device=gpu)
    accumulate_weights(q, args[1], tables, lens, offsets, lse, sums, window=200, sinks=5)
    live = lse.numel()
    assert abs(float(sums[high:].double().sum()) - live) <= live * 2.0 ** -15 and not sums[:high].any()
    # eviction moves what lies there
    before = sums.clone()
    kept = evict_tokens(sums, lens, torch.full_like(lens, 60), tables, args[1:] if bits == 4 else [tuple(args[1:])], sinks=5)
    assert kept.tolist() == [60, 60]
    for r in range(2):
        row = before[tables[r].clamp(min=0).long()].flatten()[:int(lens[r])]
        rest = row[5:].sort(descending=True, stable=True).indices[:55].sort().values + 5
        stay = torch.cat((row[:5], row[rest]))
        assert torch.equal(sums[tables[r].clamp(min=0).long()].flatten()[:60], stay)


@pytest.mark.parametrize("requests", [1, 3])
def test_many_rows_over_tables_too_wide_to_widen_together(gpu, requests):
    b = Batch(4, [200, 90, 130][:requests], [70, 66, 100][:requests], 2, 2, 128, 16, torch.float16, 4, columns=40000)
    args = b.args(gpu)
    want = b.oracle(window=100, sinks=7)
    for context in (None, 256):
        b.check(attend(b, args, window=100, sinks=7, max_context=context, return_lse=True), want)
        b.check(attend(b, args, True, window=100, sinks=7, max_context=context, return_lse=True), want)


@pytest.mark.parametrize("context", [None, 128, 40])
def test_sums_over_tables_wider_than_the_texts(gpu, context):
    """Few tokens expected of wide tables: the parts of the rows are bounded by the sums' room"""
    lens, counts = [300, 130], [120, 90]
    b = Batch(4, lens, counts, 16, 2, 128, 16, torch.bfloat16, 16, columns=60000)
    args = b.args(gpu)
    _, lse = attend(b, args, return_lse=True)
    sums = torch.zeros(b.blocks, b.bs, device=gpu)
    accumulate_weights(args[0], args[1], *args[-3:], lse, sums, max_context=context)
    given = lse.double().cpu().numpy()
    want, far = W.accumulate(np.zeros((b.blocks, b.bs), np.float32), b.q.double().numpy(), b.dense()[0], b.tables, b.lens,
                             b.offsets, given, b.dim ** -0.5, None, None, 0)
    e = (b.dim + 12) * 2.0 ** -23 * far + 2.0 ** -20 + (sum(counts) * 16 + 16) * 2.0 ** -24
    assert (np.abs(sums.double().cpu().numpy() - want) <= e * np.abs(want)).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [2, 70])
def test_other_streams(gpu, tokens, bits):
    b = batch(tokens, bits)
    args = b.args(gpu)
    want = b.oracle(window=64, sinks=4)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams * 3:
        with torch.cuda.stream(s):
            out = attend(b, args, len(outs) % 4 > 1, window=64, sinks=4, return_lse=True)
            sums = torch.zeros(b.blocks, b.bs, device=gpu)
            accumulate_weights(args[0], args[1], *args[-3:], out[1], sums, window=64, sinks=4)
            outs.append((*out, sums))
    for s in streams:
        s.synchronize()
    for out, lse, sums in outs:
        b.check((out, lse), want)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens,rows", [(1, 2), (70, 140), (70, 20000)])
def test_captured_steps(gpu, tokens, rows, bits):
    """One graph serves steps whose lengths and tables differ; two graphs on one pool take turns with
    eager work between them."""
    sets = [Batch(s, lens, counts, 16, 2, 128, 16, torch.bfloat16, bits, columns=30)
            for s, (lens, counts) in enumerate([([tokens + 300, 90], [tokens, 1]), ([tokens + 9, 400], [1, tokens]),
                                                ([tokens + 150, 200], [tokens, 0])])]
    blocks = max(b.blocks for b in sets)
    budget = torch.tensor([60, 80], dtype=torch.int32, device=gpu)

    def step(args, sums):
        out, lse = attend(sets[0], args, window=128, sinks=4, max_tokens=rows, return_lse=True)
        q, *cache, tables, lens, offsets = args
        accumulate_weights(q, cache[0], tables, lens, offsets, lse, sums, window=128, sinks=4, max_tokens=tokens)
        kept = evict_tokens(sums, lens, budget, tables, cache if bits == 4 else [tuple(cache)], sinks=4, recent=10)
        return out, lse, kept

    def state(b):
        q, *cache, tables, lens, offsets = b.args(gpu)
        q = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, rows - q.shape[0]))
        if bits == 16:
            cache = [torch.nn.functional.pad(c, (0, 0, 0, 0, 0, 0, 0, blocks - b.blocks)) for c in cache]
        else:
            big = KVCache4(blocks, 16, 2, 128, gpu)
            write_kv4(b.kc.to(gpu).flatten(0, 1), b.vc.to(gpu).flatten(0, 1), big, torch.arange(b.blocks * 16, device=gpu))
            cache = [big]
        return [q, *cache, tables, lens, offsets], torch.zeros(blocks, 16, device=gpu)

    def tensors(args, sums):
        return [t for a in args for t in (a.parts if isinstance(a, KVCache4) else [a])] + [sums]

    live, pool, graphs = [state(sets[0]) for _ in range(2)], torch.cuda.graph_pool_handle(), []
    step(*state(sets[0]))
    torch.cuda.synchronize()
    for s in live:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            got = step(*s)
        graphs.append((g, got))
    for turn in range(4):
        for i, ((g, got), s) in enumerate(zip(graphs, live)):
            b = sets[(turn + i) % 3]
            fresh, other = state(b), state(b)
            for to, x in zip(tensors(*s), tensors(*fresh)):
                to.copy_(x)
            g.replay()
            want = step(*other)  # eagerly, the same
            n = b.offsets[-1]
            assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1][:n], want[1][:n])
            assert torch.equal(got[2], want[2])
            for x, y in zip(tensors(*s), tensors(*other)):
                assert torch.equal(x, y)
            torch.cuda.synchronize()


def test_empty_calls(gpu):
    b = Batch(1, [30, 0], [0, 0], 4, 2, 64, 16, torch.bfloat16)
    args = b.args(gpu)
    out, lse = attend(b, args, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    one = torch.zeros(1, dtype=torch.int32, device=gpu)
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device=gpu)
    out = torch.full_like(q, 5.0)
    window_attention(q, *args[1:3], args[3][:0], none, one, out=out)
    assert (out == 5.0).all()
    out, lse = window_attention(q, *args[1:3], args[3][:1, :0], one, torch.tensor([0, 3], dtype=torch.int32, device=gpu),
                                return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()
    sums = torch.ones(b.blocks, 16, device=gpu)
    accumulate_weights(args[0], args[1], *args[-3:], torch.zeros(0, 4, device=gpu), sums)
    assert (sums == 1).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_refusals(gpu, bits):
    b = batch(3, bits)
    args = b.args(gpu)
    n = len(args)
    q, lens, offsets, tables = args[0], n - 2, n - 1, n - 3

    def refuse(error, change=None, **kw):
        a = list(args)
        for i, x in (change or {}).items():
            a[i] = x
        with pytest.raises(error):
            attend(b, a, **kw)
        sums = torch.zeros(b.blocks, b.bs, device=gpu)
        if "out" not in kw:
            with pytest.raises(error):
                accumulate_weights(a[0], a[1], *a[-3:], torch.zeros(q.shape[:2], device=gpu), sums, **kw)
        assert not sums.any()

    refuse(ValueError, window=0)
    refuse(ValueError, window=-4)
    refuse(ValueError, sinks=-1)
    refuse(ValueError, max_tokens=0)
    refuse(ValueError, scale=float("nan"))
    refuse(ValueError, {0: q.cpu()})
    refuse(ValueError, {lens: args[lens].cpu()})
    refuse(ValueError, {lens: args[lens][:-1]})
    refuse(ValueError, {tables: args[tables][:-1]})
    refuse(ValueError, {tables: args[tables][:, ::2]} if args[tables].shape[1] > 2 else {tables: args[tables][:-1]})
    refuse(ValueError, {offsets: args[offsets][:-1]})
    refuse(TypeError, {lens: args[lens].long()})
    refuse(TypeError, {0: q.float()})
    refuse(ValueError, {0: q[..., :64]})
    refuse(ValueError, {0: q[:, :15]})
    refuse(ValueError, {0: q[0]})
    if bits == 16:
        refuse(TypeError, {0: q.half()})
    refuse(ValueError, out=q[:-1])
    refuse(ValueError, out=q.float())
    refuse(ValueError, out=torch.empty(q.shape[0], 32, 128, dtype=q.dtype, device=gpu)[:, ::2])
    if bits == 16:
        refuse(ValueError, out=args[1].flatten()[:q.numel()].view(q.shape))
    refuse(ValueError, {0: torch.cat((q, q))[1:1 + len(q)]}, out=torch.cat((q, q))[:len(q)].cpu())
    both = torch.cat((q, q))
    refuse(ValueError, {0: both[1:1 + len(q)]}, out=both[:len(q)])


def test_refusals_of_accumulated_weights(gpu):
    b = batch(3, 16)
    q, k, v, tables, lens, offsets = b.args(gpu)
    _, lse = window_attention(q, k, v, tables, lens, offsets, return_lse=True)
    sums = torch.zeros(b.blocks, b.bs, device=gpu)

    def refuse(error, lse=lse, sums=sums, **kw):
        with pytest.raises(error):
            accumulate_weights(q, k, tables, lens, offsets, lse, sums, **kw)

    refuse(ValueError, lse=lse[:-1])
    refuse(ValueError, lse=lse.double())
    refuse(ValueError, lse=torch.zeros(len(q), 32, device=gpu)[:, ::2])
    refuse(TypeError, sums=sums.double())
    refuse(ValueError, sums=sums[:-1])
    refuse(ValueError, sums=sums.cpu())
    refuse(ValueError, sums=torch.zeros(b.bs, b.blocks, device=gpu).t())
    refuse(ValueError, new_lens=lens[:-1])
    refuse(TypeError, new_lens=lens.long())
    assert not sums.any()
