"""Weights accumulated per cached token and eviction by them, against the oracle.

A weight e^(score - lse) that is added is off by a factor of 1 + e: the score by (D + 12)
2^-23 of scale sum |q||k| (tests/bounded.py), lse log2(e) and the difference by roundings
of as much as |lse|, v_exp_f32 by a few units: e = (D + 12) 2^-23 reach + 2^-20, reach =
scale sum |q||k| + |lse|.  The additions, of at most rows * heads numbers, round by 2^-24
of the sum each."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bounded import HEADS, Batch
from oracle import window_oracle as W
from pageserve_amd import KVCache4, accumulate_weights, evict_tokens, read_kv4, write_kv4
from pageserve_amd import truncate_blocks, window_attention, window_attention4

pytestmark = pytest.mark.gpu


def accumulate(b, gpu, lse, weights, args=None, **kw):
    q, *cache, tables, lens, offsets = args or b.args(gpu)
    accumulate_weights(q, cache[0], tables, lens, offsets, lse, weights, **kw)


def check_weights(b, got, want, far, what=""):
    rows = b.offsets[-1] * b.heads
    e = (b.dim + 12) * 2.0 ** -23 * far + 2.0 ** -20 + (rows + 16) * 2.0 ** -24
    got = got.double().cpu().numpy()
    assert (np.abs(got - want) <= e * np.abs(want)).all(), what


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("tokens", [1, 3, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [16, 4])
def test_weights_of_rows(gpu, heads, tokens, dtype, bits):
    lens = [tokens, 15, 16, 17, 33, 200, 300]
    counts = [tokens] + [min(tokens, x) for x in lens[1:-1]] + [0]
    b = Batch(tokens, lens, counts, *HEADS[heads], 16, dtype, bits, garbage=float("nan"))
    args = b.args(gpu)
    start = torch.rand(b.blocks, b.bs, device=gpu)
    q = b.q.double().numpy()
    for window, sinks in ((None, 0), (20, 4), (1, 0), (100, 50)):
        lse = b.oracle(window=window, sinks=sinks)[1]
        given = torch.from_numpy(np.nan_to_num(lse)).float()
        for new in (None, [1, 0, 5, 400, 33, 7, -1]):
            want, far = W.accumulate(start.cpu().numpy(), q, b.dense()[0], b.tables, b.lens, b.offsets,
                                     given.double().numpy(), b.dim ** -0.5, new, window, sinks)
            kw = {"window": window, "sinks": sinks, "new_lens": None if new is None else b.ints(gpu, new)}
            for context in (None, 40, 10 ** 6):
                got = start.clone()
                accumulate(b, gpu, given.to(gpu), got, args, max_context=context, **kw)
                check_weights(b, got, want, far, f"{kw} {context}")
                again = start.clone()
                accumulate(b, gpu, given.to(gpu), again, args, max_context=context, max_tokens=tokens, **kw)
                assert torch.equal(got, again)


def test_weights_of_a_row_add_up_to_its_heads(gpu):
    b = Batch(5, [500, 70], [30, 70], 16, 2, 128, 16, torch.bfloat16)
    args = b.args(gpu)
    _, lse = window_attention(*args, window=64, sinks=2, return_lse=True)
    w = torch.zeros(b.blocks, b.bs, device=gpu)
    accumulate(b, gpu, lse, w, args, window=64, sinks=2)
    # (each weight within 2^-17 of its own: sums of 1 within that)
    assert abs(float(w.double().sum()) - 100 * 16) < 100 * 16 * 2.0 ** -15
    assert not w[~b.owned.to(gpu)].any()


SHAPES = [  # lens, budget, sinks, recent
    ([40, 17, 0, 5, 64], [20, 16, 3, 9, 0], 2, 3), ([1000, 999, 30], [500, 1, 30], 0, 0), ([300, 300], [100, -4], 4, 90),
    ([300, 70], [50, 60], 70, 20), ([129, 300], [128, 299], 0, 128), ([2500], [1300], 16, 200), ([33], [32], 1, 1),
]


def evict_case(gpu, lens, budget, seed, dim=128, kv=2, bs=16, bits=16, layers=2, weights=None, absent=()):
    rng = np.random.default_rng(seed)
    have = [-(-n // bs) for n in lens]
    blocks = sum(have) + 3
    order, at = rng.permutation(blocks).tolist(), 0
    tables = np.full((len(lens), max(have + [1]) + 1), -1, np.int32)
    for b, h in enumerate(have):
        tables[b, :h] = order[at:at + h]
        at += h
    for b, c in absent:
        tables[b, c] = -1
    w = np.exp(2 * rng.standard_normal((blocks, bs))).astype(np.float32) if weights is None else weights(rng, (blocks, bs))
    pairs = [[torch.from_numpy(rng.standard_normal((blocks, bs, kv, dim))).to(torch.bfloat16) for _ in range(2)]
             for _ in range(layers)]
    i = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32).to(gpu)  # noqa: E731
    caches = []
    for k, v in pairs:
        if bits == 16:
            caches.append((k.to(gpu), v.to(gpu)))
        else:
            c = KVCache4(blocks, bs, kv, dim, gpu)
            write_kv4(k.to(gpu).flatten(0, 1), v.to(gpu).flatten(0, 1), c, torch.arange(blocks * bs, device=gpu))
            caches.append(c)
    return w, tables, caches, (torch.from_numpy(w).to(gpu), i(lens), i(budget), i(tables), caches)


def contents(caches, blocks, bs, gpu):
    """The caches' rows as numpy arrays [blocks, block_size, ...]"""
    out = []
    for c in caches:
        rows = read_kv4(c, torch.arange(blocks * bs, device=gpu), torch.float32) if isinstance(c, KVCache4) else c
        out += [x.float().cpu().numpy().reshape(blocks, bs, *x.shape[-2:]) for x in rows]
    return out


@pytest.mark.parametrize("lens,budget,sinks,recent", SHAPES)
@pytest.mark.parametrize("bits,dim,bs", [(16, 128, 16), (16, 64, 48), (4, 128, 16), (4, 64, 32)])
def test_what_stays_and_where_it_goes(gpu, lens, budget, sinks, recent, bits, dim, bs):
    w, tables, caches, args = evict_case(gpu, lens, budget, sum(lens), dim, 2, bs, bits)
    before = contents(caches, *w.shape, gpu)
    want_w = w.copy()
    kept = W.evict(want_w, tables, lens, budget, before, sinks, recent)
    got = evict_tokens(*args, sinks=sinks, recent=recent, max_context=max(lens))
    assert got.tolist() == kept and got.dtype == torch.int32
    assert np.array_equal(args[0].cpu().numpy(), want_w)
    for x, y in zip(contents(caches, *w.shape, gpu), before):
        assert np.array_equal(x, y)
    assert args[1].tolist() == lens and np.array_equal(args[3].cpu().numpy(), tables)


@pytest.mark.parametrize("weights", [
    lambda rng, s: np.zeros(s, np.float32),
    lambda rng, s: rng.choice(np.float32([0.0, -0.0, 1.0, 1.5]), s),
    lambda rng, s: rng.choice(np.float32([np.nan, np.inf, -np.inf, 1e-40, -1e-40, 3.0, -3.0]), s),
    lambda rng, s: (1 + rng.integers(0, 5, s) * np.float32(2.0) ** -23).astype(np.float32),
    lambda rng, s: -np.exp(rng.standard_normal(s)).astype(np.float32),
], ids=["zeros", "ties", "special", "neighbours", "negative"])
def test_orders_of_any_numbers(gpu, weights):
    lens, budget = [700, 65, 1500], [350, 64, 100]
    w, tables, caches, args = evict_case(gpu, lens, budget, 3, layers=1, weights=weights)
    before = contents(caches, *w.shape, gpu)
    want_w = w.copy()
    kept = W.evict(want_w, tables, lens, budget, before, 3, 10)
    assert evict_tokens(*args, sinks=3, recent=10).tolist() == kept
    assert np.array_equal(args[0].cpu().numpy(), want_w, equal_nan=True)
    for x, y in zip(contents(caches, *w.shape, gpu), before):
        assert np.array_equal(x, y)


def test_absent_blocks_and_a_longer_request_than_expected(gpu):
    lens, budget = [200, 90, 300], [120, 40, 50]
    w, tables, caches, args = evict_case(gpu, lens, budget, 8, absent=[(0, 2), (0, 7), (1, 0)])
    before = contents(caches, *w.shape, gpu)
    want_w = w.copy()
    kept = W.evict(want_w, tables, lens, budget, before, 4, 8, max_context=250)
    assert kept[2] == 300
    assert evict_tokens(*args, sinks=4, recent=8, max_context=250).tolist() == kept
    assert np.array_equal(args[0].cpu().numpy(), want_w)
    for x, y in zip(contents(caches, *w.shape, gpu), before):
        assert np.array_equal(x, y)


def test_wrong_lengths_and_block_numbers_stay_inside(gpu):
    w, tables, caches, args = evict_case(gpu, [100, 64], [50, 10], 2)
    tables = args[3]
    tables[0, 3], tables[1, 1] = 1 << 30, -(1 << 31)
    kept = evict_tokens(args[0], torch.tensor([1 << 30, -5], dtype=torch.int32, device=gpu), *args[2:])
    assert kept.tolist() == [50, 0]


def test_a_cache_in_other_strides_and_many_layers(gpu):
    lens, budget = [150, 80], [64, 64]
    w, tables, caches, args = evict_case(gpu, lens, budget, 4, layers=19)
    # heads in front of slots, halves of one tensor
    moved = []
    for n, (k, v) in enumerate(caches):
        both = torch.stack((k, v), 1 if n % 3 else 4)
        if n % 3 == 1:
            both = both.transpose(2, 3).contiguous().transpose(2, 3)
        moved.append((both[:, 0], both[:, 1]) if n % 3 else (k, v))
    before = contents(caches, *w.shape, gpu)
    kept = W.evict(w.copy(), tables, lens, budget, before, 1, 2)
    assert evict_tokens(*args[:4], moved, sinks=1, recent=2).tolist() == kept
    for x, y in zip(contents(moved, *w.shape, gpu), before):
        assert np.array_equal(x, y)


@pytest.mark.parametrize("lens,budget", [([33000, 70000], [32900, 40000]), ([32768, 32769, 5], [32767, 32768, 1]),
                                         ([65000], [20])])
@pytest.mark.parametrize("bs", [16, 96])
def test_more_tokens_than_are_held_on_the_chip(gpu, lens, budget, bs):
    w, tables, caches, args = evict_case(gpu, lens, budget, 6, 64, 1, bs, layers=1)
    before = contents(caches, *w.shape, gpu)
    want_w = w.copy()
    kept = W.evict(want_w, tables, lens, budget, before, 7, 400)
    assert evict_tokens(*args, sinks=7, recent=400).tolist() == kept
    assert np.array_equal(args[0].cpu().numpy(), want_w)
    for x, y in zip(contents(caches, *w.shape, gpu), before):
        assert np.array_equal(x, y)


@pytest.mark.parametrize("heads,dim", [(3, 64), (1, 20), (2, 128)])
def test_a_cache_whose_rows_lie_at_odd_addresses(gpu, heads, dim):
    """Any size of rows at any address of two bytes."""
    lens, budget = [600, 80], [300, 64]
    w, tables, _, args = evict_case(gpu, lens, budget, 5, dim, heads, layers=0)
    rng, pair = np.random.default_rng(7), []
    for _ in range(2):
        flat = torch.from_numpy(rng.standard_normal(w.size * heads * dim + 1)).to(torch.float16).to(gpu)
        pair.append(flat[1:].view(*w.shape, heads, dim))
    before = contents([pair], *w.shape, gpu)
    kept = W.evict(w.copy(), tables, lens, budget, before, 2, 30)
    assert evict_tokens(*args[:4], [tuple(pair)], sinks=2, recent=30).tolist() == kept
    for x, y in zip(contents([pair], *w.shape, gpu), before):
        assert np.array_equal(x, y)


def test_refusals(gpu):
    w, tables, caches, args = evict_case(gpu, [40, 20], [10, 10], 1)
    weights, lens, budget, tab, _ = args
    (k, v), (k2, v2) = caches
    with pytest.raises(ValueError):
        evict_tokens(weights, lens, budget, tab, [(k, v), (k, v)])
    with pytest.raises(ValueError):
        evict_tokens(weights, lens, budget, tab, [(k, k)])
    with pytest.raises(ValueError):
        evict_tokens(weights, lens, budget, tab, [(k[:2], v[:2])])
    with pytest.raises(ValueError):
        evict_tokens(weights, lens, budget, tab, [(k, v, k2)])
    with pytest.raises(ValueError):
        evict_tokens(weights, lens, budget[:1], tab, caches)
    with pytest.raises(ValueError):
        evict_tokens(weights, lens, budget, tab, caches, sinks=-1)
    with pytest.raises(ValueError):
        evict_tokens(weights, lens, budget, tab, caches, recent=-1)
    with pytest.raises(ValueError):
        evict_tokens(weights[:, :8].contiguous(), lens, budget, tab, caches)
    with pytest.raises(TypeError):
        evict_tokens(weights.double(), lens, budget, tab, caches)
    with pytest.raises(TypeError):
        evict_tokens(weights, lens.long(), budget, tab, caches)
    with pytest.raises(TypeError):
        evict_tokens(weights, lens, budget, tab, [(k.float(), v.float())])
    with pytest.raises(RuntimeError):
        evict_tokens(weights, lens.cpu(), budget, tab, caches)
    with pytest.raises(ValueError):
        evict_tokens(weights, lens, budget, tab, [(k, k.expand(2, *k.shape)[0][:1].expand_as(k))])
    b = Batch(1, [40], [2], 2, 2, 64, 16, torch.bfloat16)
    q, kc, vc, t, n, o = b.args(gpu)
    lse, sums = torch.zeros(2, 2, device=gpu), torch.zeros(b.blocks, 16, device=gpu)
    accumulate_weights(q, kc, t, n, o, lse, sums)
    for change in ({"lse": lse[:1]}, {"lse": lse.double()}, {"weights": sums[:1]}, {"weights": sums.t()}, {"q": q[..., :32]}):
        now = {"q": q, "lse": lse, "weights": sums} | change
        with pytest.raises(ValueError):
            accumulate_weights(now["q"], kc, t, n, o, now["lse"], now["weights"])
    for kw in ({"window": 0}, {"sinks": -1}, {"max_tokens": 0}, {"scale": float("nan")}, {"new_lens": n[:0]}):
        with pytest.raises(ValueError):
            accumulate_weights(q, kc, t, n, o, lse, sums, **kw)
    with pytest.raises(TypeError):
        accumulate_weights(q.half(), kc, t, n, o, lse, sums)


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_over_what_stays(gpu, bits):
    """A whole round: rows attend, their weights are added up, requests are cut and shortened,
    and attention over the cut cache is that over the tokens that stay."""
    b = Batch(21, [180, 250, 40], [6, 1, 3], 14, 2, 64, 16, torch.bfloat16, bits, columns=18)
    q, *cache, tables, lens, offsets = b.args(gpu)
    attention = window_attention4 if bits == 4 else window_attention
    _, lse = attention(q, *cache, tables, lens, offsets, return_lse=True)
    weights = torch.full((b.blocks, b.bs), 7.0, device=gpu)
    accumulate_weights(q, cache[0], tables, lens, offsets, lse, weights, new_lens=lens)
    budget = b.ints(gpu, [100, 250, 33])
    held = weights.cpu().numpy()
    kept = evict_tokens(weights, lens, budget, tables, [cache[0] if bits == 4 else tuple(cache)], sinks=4, recent=8)
    used = [-(-n // 16) for n in b.lens]
    free, count = torch.zeros(40, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    truncate_blocks(lens, kept, tables, free, count, 16)
    assert lens.tolist() == [100, 250, 33] and int(count) == sum(used) - sum(-(-n // 16) for n in (100, 250, 33))
    got = attention(q, *cache, tables, lens, offsets, return_lse=True)
    # the oracle over the tokens that stay
    dense = b.dense()
    want = [np.zeros(s) for s in ((10, 14, 64), (10, 14), (10, 14, 64), (10, 14, 64), (10, 14))]
    for r in range(3):
        blk, at = W.places(b.tables[r], b.lens[r], 16, b.blocks)
        stay = W.stays(held[blk, at].tolist(), b.lens[r], [100, 250, 33][r], 4, 8)
        rows = slice(b.offsets[r], b.offsets[r + 1])
        few = [x[blk[stay], at[stay]][None] for x in dense]
        part = W.attention(q[rows].double().cpu().numpy(), *few, [[0]], [len(stay)], [0, rows.stop - rows.start], 0.125)
        for x, y in zip(want, part):
            x[rows] = y
    b.check(got, tuple(want), "after eviction")
