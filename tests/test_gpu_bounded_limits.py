"""Calls of the paged cache and of the operators of long texts whose grids pass what one launch may have:
2^32 threads."""

from __future__ import annotations

import pytest
import torch

from bounded import Batch
from pageserve_amd import KVCache4, accumulate_weights, evict_tokens, window_attention, window_attention4, write_kv

pytestmark = pytest.mark.gpu


def numbers(gpu, *shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu).to(dtype)


@pytest.mark.parametrize("bits,heads,dim", [(16, 8, 128), (4, 8, 64), (16, 16, 127), (16, 64, 128)])
def test_eviction_of_many_requests_in_many_layers(gpu, bits, heads, dim):
    """8192 requests x 8 heads x 16 layers and more: from 2^22 workgroups of 1024 threads on.  A few requests have tokens; the
    call gives what one of those alone gives."""
    requests, layers, bs, live, lens = 8192, 16, 16, [0, 1, 4095, 8190, 8191], [50, 16, 300, 47, 33]
    have = [-(-n // bs) for n in lens]
    blocks = sum(have) + 1
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    tables, all_lens = torch.full((requests, max(have)), -1, dtype=torch.int32), torch.zeros(requests, dtype=torch.int32)
    at = 0
    for b, n, h in zip(live, lens, have):
        tables[b, :h], all_lens[b] = order[at:at + h], n
        at += h
    budget = torch.full((requests,), 20, dtype=torch.int32)
    weights = numbers(gpu, blocks, bs, dtype=torch.float32)
    caches = []
    for i in range(layers):
        if bits == 16:
            caches.append(tuple(numbers(gpu, blocks, bs, heads, dim, seed=2 * i + j) for j in range(2)))
        else:
            c = KVCache4(blocks, bs, heads, dim, gpu)
            for j, p in enumerate(c.parts):
                p.copy_((numbers(gpu, *p.shape, dtype=torch.float32, seed=4 * i + j) * 1000).to(p.dtype))
            caches.append(c)

    def parts(caches):
        return [p for c in caches for p in (c.parts if bits == 4 else c)]

    def copy(caches):
        return [KVCache4.of(*(p.clone() for p in c.parts)) if bits == 4 else tuple(p.clone() for p in c) for c in caches]

    def call(rows, weights, caches):
        return evict_tokens(weights, all_lens[rows].to(gpu), budget[rows].to(gpu), tables[rows].to(gpu), caches, sinks=2, recent=3)

    want_weights, want = weights.clone(), copy(caches)
    before = copy(caches)
    assert call(live, want_weights, want).tolist() == [20, 16, 20, 20, 20]
    assert not all(torch.equal(x, y) for x, y in zip(parts(want), parts(before)))
    kept = call(list(range(requests)), weights, caches)
    assert torch.equal(kept.cpu(), torch.minimum(all_lens, budget))
    assert torch.equal(weights, want_weights)
    for x, y in zip(parts(caches), parts(want)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens", [1, 40])
def test_sums_of_many_requests_over_wide_tables(gpu, tokens, bits):
    """1024 requests of tables for 2^21 tokens: 2^24 workgroups of 256 threads.  Some have tokens; the call
    gives what the same call for shorter texts gives."""
    requests, bs, columns, live, lens = 1024, 65536, 32, [0, 7, 1000, 1023], [300, 41, 129, 40]
    blocks = len(live) + 1
    tables = torch.full((requests, columns), -1, dtype=torch.int32)
    all_lens, counts = torch.zeros(requests, dtype=torch.int32), torch.zeros(requests, dtype=torch.int32)
    for i, (b, n) in enumerate(zip(live, lens)):
        tables[b, 0], all_lens[b], counts[b] = blocks - 1 - i, n, tokens
    offsets = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
    q = numbers(gpu, int(offsets[-1]), 4, 64)
    if bits == 16:
        cache = tuple(numbers(gpu, blocks, bs, 1, 64, seed=i + 1) for i in range(2))
    else:
        c = KVCache4(blocks, bs, 1, 64, gpu)
        c.k.random_(), c.v.random_(), c.k_scale.fill_(0.25), c.v_scale.fill_(0.5)
        cache = (c,)
    rest = [x.to(gpu) for x in (tables, all_lens, offsets)]
    attend = window_attention if bits == 16 else window_attention4
    _, lse = attend(q, *cache, *rest, max_tokens=tokens, max_context=1000, return_lse=True)
    sums, want = torch.zeros(blocks, bs, device=gpu), torch.zeros(blocks, bs, device=gpu)
    accumulate_weights(q, cache[0], *rest, lse, sums, max_tokens=tokens)
    accumulate_weights(q, cache[0], *rest, lse, want, max_tokens=tokens, max_context=1000)
    assert torch.equal(sums, want)
    rows = lse.numel()  # (each row's weights add up to 1, each within 2^-17 of its own)
    assert abs(float(sums.double().sum()) - rows) <= rows * 2.0 ** -15


def test_many_rows_over_a_table_for_a_very_long_text_in_4_bits(gpu):
    """2^28 tokens and more: as many sixteens to widen as make 2^24 workgroups of 256 threads, 69 GB of room"""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of free memory")
    b = Batch(5, [70000], [80], 2, 1, 64, 65536, torch.bfloat16, 4, columns=4097)
    args = b.args(gpu)
    b.check(window_attention4(*args, window=300, sinks=9, return_lse=True), b.oracle(window=300, sinks=9))
    torch.cuda.empty_cache()
    b.check(window_attention4(*args, return_lse=True), b.oracle())
    torch.cuda.empty_cache()


@pytest.mark.parametrize("aligned", [False, True])
def test_rows_beyond_one_launch_of_write_kv(gpu, aligned):
    """2^32 pieces and more (of one number where something is not aligned, else of eight): the last rows too"""
    dim, bs, rows = (256, 16, (1 << 24) + 300) if not aligned else (1024, 16, (1 << 25) + 300)
    buffer = numbers(gpu, 2, dim + 8)
    k, v = (x[8 if aligned else 1:][:dim].expand(rows, 1, dim) for x in buffer)
    cache = [torch.zeros(4, bs, 1, dim, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    slots = torch.full((rows,), -1, dtype=torch.int64, device=gpu)
    slots[0], slots[(1 << 24) - 1], slots[-1] = 3, 20, 37
    write_kv(k, v, *cache, slots)
    for part, x in zip(cache, (k, v)):
        want = torch.zeros_like(part)
        want.view(-1, dim)[[3, 20, 37]] = x[0, 0]
        assert torch.equal(part, want)


@pytest.mark.parametrize("bits", [16, 4])
def test_a_step_of_many_requests_that_says_nothing_of_its_rows(gpu, bits):
    """8192 requests of one row: by default planned as if each could have all 8192"""
    lens = [1 + 7 * b % 40 for b in range(8192)]
    b = Batch(8, lens, [1] * 8192, 16, 1, 64, 16, torch.bfloat16, bits, garbage=float("nan"))
    args, want = b.args(gpu), b.oracle(window=20, sinks=2)
    attend = window_attention if bits == 16 else window_attention4
    for most in (None, 1):
        b.check(attend(*args, window=20, sinks=2, max_tokens=most, return_lse=True), want, f"max_tokens={most}")
